"""The operators of the 8-bit mixture-of-experts feed-forward, and what they are timed on.

Four of them, in the order in which a layer calls them:

  norm      the residual stream takes a sublayer's result; up to two RMS norms of the sum leave in e4m3 with a scale for
            every 128 channels of a row, the second one, where asked, in the activation type as well (a router reads that)
  linear    x w^T of such rows and a weight in e4m3 with a scale for every block of 128 x 128
  route     scores of the experts (softmax or sigmoid), a bias for the choice alone, groups of experts of which some are
            left, the k best, their weights; and the tokens in the order of their experts
  experts   route, then every expert's gelu-gated feed-forward on its tokens, in e4m3, and the weighted sum of a token's k results

A case is a dict of plain values:
  op        norm | linear | route | experts
  norm      rows, width, norms (1 or 2), plain (the last norm also in the activation type), dtype (of the sublayer's result, the weights)
  linear    rows, n, k, dtype (of the result)
  route     tokens, experts, top_k, score, bias, groups, top_groups, renormalize
  experts   tokens, width, ff and what route takes

The plain forms compute in 32 bits (the choice of experts in 64) and round once.
"""

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128                   # channels, or rows and columns of a weight, that share a scale
TOP = 448.0                   # the largest e4m3 value
LEAST = 2.0 ** -126           # the smallest scale
EPS = 1e-6


def norm(name, rows, width, norms=2, plain=False, dtype="bfloat16"):
    return dict(name=name, op="norm", rows=rows, width=width, norms=norms, plain=plain, dtype=dtype)


def linear(name, rows, n, k, dtype="bfloat16"):
    return dict(name=name, op="linear", rows=rows, n=n, k=k, dtype=dtype)


def routing(tokens, experts, top_k, score="softmax", bias=False, groups=1, top_groups=1, renormalize=True):
    return dict(tokens=tokens, experts=experts, top_k=top_k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalize=renormalize)


def route(name, *a, **kw):
    return dict(name=name, op="route", **routing(*a, **kw))


def experts(name, tokens, width, ff, n, top_k, **kw):
    return dict(name=name, op="experts", width=width, ff=ff, **routing(tokens, n, top_k, **kw))


def listed():
    return [
        # a decoding step of eight sequences at the 2048 wide model: both norms of a layer
        norm("norm_step", 8, 2048),
        # a short fp32 prompt at a width that fills no block
        norm("norm_odd_fp32", 333, 1000, dtype="float32"),
        # a server's step of prompts: one norm for the mixer, one for router and experts
        norm("norm_prompt", 32768, 2048, plain=True),
        # the projection of a feed-forward while four sequences decode
        linear("linear_step", 4, 8192, 2048),
        # odd sizes everywhere, a few dozen rows
        linear("linear_odd_fp32", 77, 1000, 1304, dtype="float32"),
        # one prompt through the narrow model's feed-forward
        linear("linear_prompt", 3000, 8192, 1024),
        # a full step of prompts through the wide model's projection
        linear("linear_large", 16384, 8192, 4096),
        # a decoding step's choice of experts
        route("route_step", 8, 64, 8),
        # the choice of a step of prompts: many experts in groups, balanced by a bias
        route("route_prompt", 16384, 256, 8, score="sigmoid", bias=True, groups=8, top_groups=4),
        # sixteen sequences decode: most experts have a token or two
        experts("experts_step", 16, 2048, 1024, 64, 8),
        # a short prompt at sizes that fill no block, a few experts
        experts("experts_odd", 300, 720, 200, 10, 2, score="sigmoid", renormalize=False),
        # a step of prompts
        experts("experts_prompt", 8192, 2048, 1024, 64, 8, score="sigmoid", bias=True, groups=8, top_groups=4),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)

    def choice(n, tokens):
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if n % g == 0 and n // g >= 2] or [1])
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, n // groups * top_groups))
        return routing(tokens, n, k, rng.choice(("softmax", "sigmoid")), rng.random() < 0.5, groups, top_groups, rng.random() < 0.7)

    op = rng.choice(("norm", "linear", "linear", "route", "experts"))
    if op == "norm":
        width = size(64, 8192, rng.choice((1, 4, 128)))
        norms = rng.choice((1, 2))
        return dict(op=op, rows=min(size(1, 32768), 32768 * 2048 // width), width=width, norms=norms, plain=rng.random() < 0.4,
                    dtype=rng.choice(("bfloat16", "bfloat16", "float32")))
    if op == "linear":
        n, k = size(16, 16384, rng.choice((1, 8, 128))), size(16, 8192, rng.choice((1, 8, 128)))
        return dict(op=op, rows=min(size(1, 16384), 16384 * 8192 * 4096 // (n * k)), n=n, k=k, dtype=rng.choice(("bfloat16", "bfloat16", "float32")))
    if op == "route":
        n = rng.choice((size(2, 512), size(1, 64) * 8))
        return dict(op=op, **choice(n, min(size(1, 65536), 16384 * 256 // n)))
    n = rng.choice((size(2, 64), size(1, 8) * 8))
    width, ff = size(64, 4096, rng.choice((1, 8, 128))), size(64, 2048, rng.choice((1, 8, 128)))
    while n * width * ff > 64 * 2048 * 1024:
        n = max(2, n // 2)
    c = choice(n, 1)
    c["tokens"] = min(size(1, 8192), 8192 * 8 * 2048 * 1024 // (c["top_k"] * width * ff))
    return dict(op=op, width=width, ff=ff, **c)


# ---- inputs --------------------------------------------------------------------------------------------------------------
def blocks(n):
    return -(-n // BLOCK)


def dtype_of(case):
    return getattr(torch, case["dtype"])


def padded(rows, cols):
    """Storage for e4m3 rows that start on 16-byte boundaries."""
    return torch.zeros(*rows, -(-cols // 16) * 16, device=DEV, dtype=torch.float8_e4m3fn)[..., :cols]


def e4m3_rows(x):
    """(values, scales) of rows in 8 bits; the scales lie block by block."""
    rows, cols = x.shape
    nb = blocks(cols)
    xb = torch.zeros(rows, nb * BLOCK, device=DEV)
    xb[:, :cols] = x
    xb = xb.view(rows, nb, BLOCK)
    s = (xb.abs().amax(-1) / TOP).clamp_min(LEAST)
    values = padded((rows,), cols)
    values.copy_((xb / s[..., None]).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn))
    scales = torch.empty(nb, rows, device=DEV).t()
    return values, scales.copy_(s)


def e4m3_weight(gen, *shape):
    """(values, scales) of a random weight (..., N, K) in 8 bits with a scale for each block of 128 x 128."""
    *lead, n, k = shape
    count = math.prod(lead)
    nb, kb = blocks(n), blocks(k)
    values, scales = padded((count, n), k), torch.empty(count, nb, kb, device=DEV)
    for i in range(count):
        w = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
        w[:n, :k] = torch.randn(n, k, device=DEV, generator=gen) * k ** -0.5
        wb = w.view(nb, BLOCK, kb, BLOCK)
        s = (wb.abs().amax((1, 3)) / TOP).clamp_min(LEAST)
        values[i].copy_((wb / s[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn))
        scales[i] = s
    return values.unflatten(0, lead) if lead else values[0], scales.view(*lead, nb, kb)


def activations(gen, rows, width):
    """Rows with a few channels far above the others, as a residual stream has them."""
    x = torch.randn(rows, width, device=DEV, generator=gen)
    loud = torch.rand(width, device=DEV, generator=gen) < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def prepare_routing(case, gen):
    n = case["experts"]
    logits = 1.5 * torch.randn(case["tokens"], n, device=DEV, generator=gen) + 0.5 * torch.randn(n, device=DEV, generator=gen)
    return dict(logits=logits, bias=0.1 * torch.randn(n, device=DEV, generator=gen) if case["bias"] else None)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "norm":
        rows, width, dtype = case["rows"], case["width"], dtype_of(case)
        st["x"] = activations(gen, rows, width)
        st["y"] = torch.randn(rows, width, device=DEV, generator=gen).to(dtype)
        st["weights"] = [(0.1 * torch.randn(width, device=DEV, generator=gen)).to(dtype) for _ in range(case["norms"])]
        st["sum"] = torch.empty_like(st["x"])
    elif case["op"] == "linear":
        st["x"], st["xs"] = e4m3_rows(activations(gen, case["rows"], case["k"]))
        st["w"], st["ws"] = e4m3_weight(gen, case["n"], case["k"])
    else:
        st.update(prepare_routing(case, gen))
        if case["op"] == "experts":
            n, width, ff = case["experts"], case["width"], case["ff"]
            st["h"] = activations(gen, case["tokens"], width).bfloat16()
            st["w_in"], st["w_in_s"] = e4m3_weight(gen, n, 2, ff, width)
            st["w_out"], st["w_out_s"] = e4m3_weight(gen, n, width, ff)
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------------------
def rounded(x):
    """fp64 values up to 448 to the nearest e4m3 one, ties to the even one (a conversion would round to fp32 in between)."""
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x).exponent.clamp_min(-5) - 4)
    return (torch.round(x / step) * step).to(torch.float8_e4m3fn)


def quantized(x):
    """(values, scales, what they stand for) of fp32 rows (..., width).  The quotients are 64 bits wide: 16-bit values over a largest
    one of them lie on borders between two e4m3 values in numbers."""
    width = x.shape[-1]
    xb = torch.nn.functional.pad(x, (0, blocks(width) * BLOCK - width)).unflatten(-1, (-1, BLOCK))
    s = torch.clamp(xb.abs().amax(-1).double() / TOP, min=LEAST).float()
    q = rounded(xb.double() / s[..., None].double())
    meant = q.float() * s[..., None]
    return q.flatten(-2)[..., :width], s, meant.flatten(-2)[..., :width]


def widened(values, scales):
    """A weight (..., N, K) in fp32."""
    n, k = values.shape[-2:]
    s = scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return values.float() * s


def gelu(z):
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def plain_norm(st):
    case, x = st["case"], st["x"] + st["y"].float()
    unit = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    out = [x]
    for i, w in enumerate(st["weights"]):
        h = unit * (1 + w.float())
        out += quantized(h)[:2]
        if case["plain"] and i == len(st["weights"]) - 1:
            out.append(h.to(dtype_of(case)))
    return out


def best(keys, k):
    """The k largest of every row in falling order, of equal ones the lowest index first."""
    return torch.sort(keys, dim=-1, descending=True, stable=True).indices[..., :k]


def plain_route(st):
    case = st["case"]
    tokens, n, k, groups = case["tokens"], case["experts"], case["top_k"], case["groups"]
    logits = st["logits"].double()
    score = torch.sigmoid(logits) if case["score"] == "sigmoid" else torch.softmax(logits, -1)
    if st["bias"] is None and groups == 1:
        keys = logits                                                      # both scores grow with it
    else:
        keys = score if st["bias"] is None else score + st["bias"].double()
    if groups > 1:
        of_group = torch.sort(keys.view(tokens, groups, -1), dim=-1, descending=True).values[..., :2].sum(-1)
        left = torch.zeros(tokens, groups, device=DEV, dtype=torch.bool).scatter_(1, best(of_group, case["top_groups"]), True)
        keys = torch.where(left.repeat_interleave(n // groups, 1), keys, -math.inf)
    ids = best(keys, k)
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    order = torch.sort(ids.flatten(), stable=True).indices
    starts = torch.searchsorted(ids.flatten()[order], torch.arange(n + 1, device=DEV))
    return ids.int(), weights.float(), order.int(), starts.int()


def plain_experts(st):
    case = st["case"]
    tokens, n, k, width, ff = case["tokens"], case["experts"], case["top_k"], case["width"], case["ff"]
    ids, weights, order, starts = plain_route(st)
    order, starts = order.long(), starts.long()
    of = ids.flatten().long()[order]                                       # expert of every row, and its place among the expert's
    place = torch.arange(tokens * k, device=DEV) - starts[of]
    x = torch.zeros(n, int((starts[1:] - starts[:-1]).max()), width, device=DEV)
    x[of, place] = quantized(st["h"].float())[2][order // k]
    z = x @ widened(st["w_in"], st["w_in_s"]).flatten(1, 2).transpose(1, 2)
    a = quantized(gelu(z[..., :ff]) * z[..., ff:])[2]
    y = a @ widened(st["w_out"], st["w_out_s"]).transpose(1, 2)
    back = torch.empty(tokens * k, width, device=DEV)
    back[order] = y[of, place]
    return (back.view(tokens, k, width) * weights[..., None]).sum(1).bfloat16()


def plain(st):
    op = st["case"]["op"]
    if op == "norm":
        return plain_norm(st)
    if op == "linear":
        x = st["x"].float() * st["xs"].repeat_interleave(BLOCK, 1)[:, :st["case"]["k"]]
        return (x @ widened(st["w"], st["ws"]).t()).to(dtype_of(st["case"]))
    return plain_route(st) if op == "route" else plain_experts(st)


# ---- the framework's ------------------------------------------------------------------------------------------------------
def routes_of(st):
    from atma_b200.experts import route_experts
    c = st["case"]
    return route_experts(st["logits"], c["top_k"], score=c["score"], bias=st["bias"], groups=c["groups"], top_groups=c["top_groups"],
                         renormalize=c["renormalize"])


def framework(st):
    from atma_b200 import fp8_ops
    case, op = st["case"], st["case"]["op"]
    if op == "norm":
        normed = fp8_ops.residual_norms_fp8(st["x"], st["y"], st["weights"], EPS, out=st["sum"], plain=case["plain"])
        return [st["sum"]] + [t for rows, h in normed for t in (rows.values, rows.scales, h) if t is not None]
    if op == "linear":
        return fp8_ops.linear_fp8(fp8_ops.Fp8Rows(st["x"], st["xs"]), fp8_ops.Fp8Weight(st["w"], st["ws"]), dtype=dtype_of(case))
    routes = routes_of(st)
    if op == "route":
        return routes.ids, routes.weights, routes.order, routes.starts
    from atma_b200.experts import expert_mlp
    return expert_mlp(fp8_ops.quantize_rows(st["h"]), fp8_ops.Fp8Weight(st["w_in"], st["w_in_s"]), fp8_ops.Fp8Weight(st["w_out"], st["w_out_s"]),
                      routes, dtype=torch.bfloat16)


def run(state):
    return framework(state) if own else plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["width"], 2 if case["dtype"] == "bfloat16" else 4
        scales = 4 * case["rows"] * blocks(case["width"])
        return {"bytes": n * (4 + size + 4) + case["norms"] * (n + scales) + (n * size if case["plain"] else 0), "flops": 8 * n}
    if case["op"] == "linear":
        m, n, k, size = case["rows"], case["n"], case["k"], 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": m * k + n * k + m * n * size + 4 * blocks(k) * (m + blocks(n)), "flops": 2 * m * n * k}
    t, n, k = case["tokens"], case["experts"], case["top_k"]
    nbytes = 4 * t * n + 12 * t * k + 4 * (n + 1)
    if case["op"] == "route":
        return {"bytes": nbytes, "flops": 8 * t * n}
    width, ff = case["width"], case["ff"]
    called = n * (1 - (1 - k / n) ** t)                                    # experts with a token, where all are as likely
    return {"bytes": int(nbytes + 4 * t * width + called * 3 * width * ff), "flops": 6 * t * k * width * ff}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact_scale(cells):
    """Scales are fp32 values by definition."""
    return torch.maximum(cells.abs().max(-1).values / 448, torch.tensor(2.0 ** -126, device=DEV, dtype=torch.float64)).float().double()


def exact_e4m3(x):
    """By the table of all values and the borders between them."""
    table = torch.arange(127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    borders = (table[1:] + table[:-1]) / 2
    at = torch.searchsorted(borders, x.abs().contiguous())                                # on a border: the lower one
    on = x.abs() == borders[at.clamp_max(125)]
    at = torch.where(on & (at % 2 == 1), at + 1, at)
    return table[at] * x.sign()


def exact_rows(x):
    """(scales, e4m3 values) of fp64 rows, block by block."""
    scales, values = [], []
    for c in range(0, x.shape[1], 128):
        s = exact_scale(x[:, c:c + 128])
        scales.append(s)
        values.append(exact_e4m3(x[:, c:c + 128] / s[:, None]))
    return torch.stack(scales, 1), torch.cat(values, 1)


def exact_product(x, xs, w, ws):
    """sum over blocks of columns of xs ws (x w^T), everything fp64."""
    out = torch.zeros(x.shape[0], w.shape[0], device=DEV, dtype=torch.float64)
    for b, c in enumerate(range(0, x.shape[1], 128)):
        columns = ws[:, b].double().repeat_interleave(128)[:w.shape[0]]
        out += (x[:, c:c + 128] @ w[:, c:c + 128].double().t()) * xs[:, b:b + 1].double() * columns
    return out


def exact_choice(case, st):
    z = st["logits"].double()
    if case["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.max(1, keepdim=True).values)
        score = e / e.sum(1, keepdim=True)
    keys = score + (0 if st["bias"] is None else st["bias"].double())
    size = case["experts"] // case["groups"]
    if case["groups"] > 1:
        totals = torch.stack([keys[:, g * size:(g + 1) * size].topk(min(2, size), dim=1).values.sum(1) for g in range(case["groups"])], 1)
        kept = totals.topk(case["top_groups"], dim=1).indices
        out = torch.ones_like(keys, dtype=torch.bool)
        for j in range(case["top_groups"]):
            cols = kept[:, j:j + 1] * size + torch.arange(size, device=DEV)
            out.scatter_(1, cols, False)
        keys = keys.masked_fill(out, -math.inf)
    ids = keys.topk(case["top_k"], dim=1).indices
    picked = score.gather(1, ids)
    return ids, picked / picked.sum(1, keepdim=True) if case["renormalize"] else picked


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        x = st["x"].double() + st["y"].double()
        out = [x]
        for i, w in enumerate(st["weights"]):
            h = x * (x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPS).rsqrt() * (1 + w.double())
            s, q = exact_rows(h)
            out += [q, s]
            if case["plain"] and i + 1 == case["norms"]:
                out.append(h)
        return out
    if case["op"] == "linear":
        return exact_product(st["x"].double(), st["xs"], st["w"], st["ws"])
    ids, weights = exact_choice(case, st)
    if case["op"] == "route":
        return None, weights, None, None
    s, q = exact_rows(st["h"].double())
    y = torch.zeros(case["tokens"], case["width"], device=DEV, dtype=torch.float64)
    for e in range(case["experts"]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if len(t):
            gate, up = (exact_product(q[t], s[t], st["w_in"][e, i], st["w_in_s"][e, i]) for i in (0, 1))
            a = 0.5 * gate * (1 + torch.tanh((2 / math.pi) ** 0.5 * (gate + 0.044715 * gate * gate * gate))) * up
            a_s, a_q = exact_rows(a)
            y[t] += weights[t, j, None] * exact_product(a_q, a_s, st["w_out"][e], st["w_out_s"][e])
    return y
