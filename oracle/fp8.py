"""Plain 64-bit restatement of the operators in 8 bits and of the experts' routing.  TEST INFRASTRUCTURE ONLY.

No shared code with the product path; fp64 tensors, loops where the definitions have them.
"""

import math

import torch

BLOCK = 128


def e4m3_values():
    """The finite values of e4m3 from zero up, by its definition: 4 bits of exponent with bias 7, 3 of mantissa, no infinity."""
    return torch.tensor([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:-1], dtype=torch.float64)


def borders():
    v = e4m3_values()
    return (v[1:] + v[:-1]) / 2


def to_e4m3(x):
    """Nearest e4m3 value, ties to the even one, in fp64."""
    v, b = e4m3_values(), borders()
    at = torch.searchsorted(b, x.abs().contiguous())
    tie = x.abs() == b[at.clamp_max(len(b) - 1)]
    return v[torch.where(tie & (at % 2 == 1), at + 1, at)] * x.sign()


def step_at(x):
    """Distance of the e4m3 values around x."""
    return torch.ldexp(torch.ones_like(x), (torch.frexp(x).exponent - 1).clamp_min(-6) - 3)


def quantize(x):
    """(values, scales) of fp64 rows: values (rows, width) as fp64, scales (rows, blocks) rounded to fp32, as fp64."""
    q, s = torch.zeros_like(x), torch.zeros(x.shape[0], -(-x.shape[1] // BLOCK), dtype=torch.float64)
    for b in range(s.shape[1]):
        c = slice(b * BLOCK, min((b + 1) * BLOCK, x.shape[1]))
        s[:, b] = (x[:, c].abs().amax(1) / 448).clamp_min(2.0 ** -126).float().double()
        q[:, c] = to_e4m3(x[:, c] / s[:, b:b + 1])
    return q, s


def wide_rows(q, s):
    return q.double() * s.double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def wide_weight(q, s):
    """One matrix (N, K) with scales by blocks of 128 x 128."""
    return q.double() * s.double().repeat_interleave(BLOCK, 0)[:q.shape[0]].repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def norm(t, weight, eps, offset):
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps) * (offset + weight)


def gelu_tanh(z):
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(ids, weights) as lists of lists, a token at a time."""
    ids, weights = [], []
    top = torch.finfo(torch.float32).max
    for row in logits.double().tolist():
        z = [-top if math.isnan(v) else min(max(v, -top), top) for v in row]
        n, m = len(z), max(z)
        if score == "sigmoid":
            s = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in z]
        else:
            e = [math.exp(max(v - m, -1e4)) for v in z]
            s = [v / sum(e) for v in e]
        key = list(z) if bias is None and groups == 1 else [s[i] + (0.0 if bias is None else float(bias[i])) for i in range(n)]
        if groups > 1:
            size = n // groups
            two = [sorted(key[g * size:(g + 1) * size], reverse=True)[:2] for g in range(groups)]
            of = [t[0] if t[0] == math.inf else sum(t) for t in two]
            kept = sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups]
            left = [i for i in range(n) if i // size in kept]                        # also where a bias leaves their keys at -inf
        else:
            left = range(n)
        best = sorted(left, key=lambda i: (-key[i], i))[:top_k]
        w = [s[i] for i in best]
        if renormalize:
            w = [v / sum(w) if sum(w) > 0 else 0.0 for v in w]
        ids.append(best)
        weights.append([v * scale for v in w])
    return ids, weights


def order(ids, experts):
    """(order, place, starts) of a routing's pairs."""
    pairs = sorted(((e, t * len(row) + j) for t, row in enumerate(ids) for j, e in enumerate(row)))
    by = [p for _, p in pairs]
    place = [0] * len(by)
    for r, p in enumerate(by):
        place[p] = r
    return by, place, [sum(e < x for e, _ in pairs) for x in range(experts + 1)]


def expert_mlp(x, w_gate_up, w_down, ids, weights, err=0.0):
    """sum over a token's experts of weight * down(8 bits of (gelu(gate x) * up x)), and how far a result may be off if every product in
    front of the activations is off by up to ``err`` (|x| |w|^T): what that does to scales, and the steps of values that it may move
    over a border.  x (tokens, width), w_gate_up[e] = (gate, up), w_down[e]: fp64 matrices."""
    tokens, width = x.shape
    out, off, most = (torch.zeros(tokens, width, dtype=torch.float64) for _ in range(3))
    for t in range(tokens):
        for e, w in zip(ids[t], weights[t]):
            gate, up = (x[t] @ m.t() for m in w_gate_up[e])
            eg, eu = (err * (x[t].abs() @ m.abs().t()) for m in w_gate_up[e])
            a = gelu_tanh(gate) * up
            ea = 1.13 * eg * (up.abs() + eu) + (gelu_tanh(gate).abs() * eu) + 2e-5 * a.abs() * (err > 0)
            q, s = quantize(a[None])
            wide = s.repeat_interleave(BLOCK, 1)[0, :a.shape[0]]
            es = torch.stack([(ea[b * BLOCK:(b + 1) * BLOCK].max() / 448 + 2.0 ** -24 * s[0, b]) for b in range(s.shape[1])])
            es = es.repeat_interleave(BLOCK)[:a.shape[0]] * (err > 0)
            ratio = a / wide
            eq = (ea + ratio.abs() * es) / wide
            b = borders()
            at = torch.searchsorted(b, ratio.abs().contiguous()).clamp_max(len(b) - 1)
            near = torch.minimum((ratio.abs() - b[at]).abs(), (ratio.abs() - b[(at - 1).clamp_min(0)]).abs()) <= eq
            moved = torch.where(near, step_at(q[0].abs() * 1.07) * wide + es, torch.zeros_like(a)) + q[0].abs() * es
            y = (q[0] * wide) @ w_down[e].t()
            out[t] += w * y
            most[t] += abs(w) * y.abs()
            off[t] += abs(w) * (moved @ w_down[e].abs().t() + err * (q[0].abs() * wide) @ w_down[e].abs().t())
    return out, off, most


# ---- a Rizurax layer whose projections are in 8 bits, or whose feed-forward is a mixture of experts ------------------------
def round_rows(x):
    """What rows stand for after they have been in 8 bits."""
    return wide_rows(*quantize(x))


def round_weight(w):
    """What a matrix stands for after it has been in 8 bits with scales by blocks of 128 x 128."""
    out = torch.zeros_like(w)
    for i in range(0, w.shape[0], BLOCK):
        for j in range(0, w.shape[1], BLOCK):
            cell = w[i:i + BLOCK, j:j + BLOCK]
            s = (cell.abs().max() / 448).clamp_min(2.0 ** -126).float().double()
            out[i:i + BLOCK, j:j + BLOCK] = to_e4m3(cell / s) * s
    return out


def rizurax_layer(x, w, i, entry, eps, in_8_bits):
    from . import rizurax as R
    p, mix, mlp = f"l{i}.", entry["mixer"], entry.get("mlp")
    rows, weight = (round_rows, round_weight) if in_8_bits else (lambda t: t, lambda t: t)
    names = [p + "mix." + n for n in (("q", "k", "v", "g", "a", "b") if entry["type"] == "delta" else ("q", "k", "v"))]
    parts = weight(torch.cat([w[n] for n in names])).split([w[n].shape[0] for n in names])          # one matrix, whose blocks span its parts
    mixer = {"delta": R.delta_mixer, "attention": R.attention_mixer}[entry["type"]]
    size = w[p + "mix.o"].shape[1]
    inner = {**w, **dict(zip(names, parts)), p + "mix.o": torch.eye(size, dtype=x.dtype)}
    out = x + rows(mixer(rows(R.rms_norm_centered(x, w[p + "norm1"], eps)), inner, p + "mix.", mix, eps)) @ weight(w[p + "mix.o"]).T
    if mlp is None:
        return out
    h = R.rms_norm_centered(x, w[p + "norm2"], eps)
    gate, up, down = (w[p + "mlp." + n] for n in ("gate", "up", "down"))
    if mlp.get("kind", "dense") == "dense":
        a = R.gelu_tanh(rows(h) @ weight(gate).T) * (rows(h) @ weight(up).T)
        return out + rows(a) @ weight(down).T
    ids, weights = route(h @ w[p + "mlp.router"].T, mlp["top_k"], mlp.get("score", "softmax"), w[p + "mlp.router.bias"] if mlp.get("bias") else None,
                         mlp.get("groups", 1), mlp.get("top_groups") or mlp.get("groups", 1), mlp.get("renormalize", True), mlp.get("scale", 1.0))
    both = [(round_weight(g), round_weight(u)) for g, u in zip(gate, up)]
    return out + expert_mlp(round_rows(h), both, [round_weight(d) for d in down], ids, weights)[0]


def rizurax_forward(cfg, w, tokens):
    """Logits (T, vocab) of one sequence."""
    from . import rizurax as R
    w = {n: t.double() for n, t in w.items()}
    eps, x = cfg["norm"]["eps"], R.embed(tokens, w, cfg["embedding"].get("bigram"))
    for i in R.layer_order(cfg):
        x = rizurax_layer(x, w, i, cfg["layers"][i], eps, cfg.get("weights") == "e4m3")
    return R.rms_norm_centered(x, w["final.norm"], eps) @ w["head"].T


def rizurax_weights(cfg, seed):
    """``oracle.rizurax.random_weights`` with the experts' tensors."""
    from . import rizurax as R
    plain = {**cfg, "layers": [{**e, "mlp": None if (e.get("mlp") or {}).get("kind") == "experts" else e.get("mlp")} for e in cfg["layers"]]}
    w, g, D = R.random_weights(plain, seed), torch.Generator().manual_seed(1000 + seed), cfg["width"]
    put = lambda name, *shape, std=None: w.__setitem__(name, (torch.randn(*shape, generator=g) * (shape[-1] ** -0.5 if std is None else std)).bfloat16().float())
    for i, e in enumerate(cfg["layers"]):
        m, p = e.get("mlp") or {}, f"l{i}."
        if m.get("kind") == "experts":
            put(p + "norm2", D, std=0.2)
            put(p + "mlp.router", m["experts"], D)
            if m.get("bias"):
                put(p + "mlp.router.bias", m["experts"], std=0.1)
            put(p + "mlp.gate", m["experts"], m["ff"], D)
            put(p + "mlp.up", m["experts"], m["ff"], D)
            put(p + "mlp.down", m["experts"], D, m["ff"])
    return w
