"""GPU: routing to experts and their feed-forwards in 8 bits, against fp64 (oracle/fp8.py)."""

import math

import pytest
import torch

from oracle import fp8 as O
from tests.test_gpu_fp8 import loud, ops, product_error, rand, weight8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def routing():
    from atma_b200 import experts
    return experts


def check_order(r):
    by, place, starts = O.order(r.ids.tolist(), r.experts)
    assert r.order.tolist() == by and r.place.tolist() == place and r.starts.tolist() == starts


ROUTES = [(1, 2, 1, {}), (5, 8, 2, {}), (3, 1, 1, {}), (40, 10, 3, dict(score="sigmoid")), (129, 64, 8, {}), (200, 33, 5, dict(bias=True)),
          (300, 65, 4, dict(bias=True, score="sigmoid", renormalize=False, scale=2.5)), (150, 256, 8, dict(bias=True, score="sigmoid", groups=8, top_groups=4)),
          (70, 96, 6, dict(groups=6, top_groups=2)), (64, 40, 7, dict(groups=40, top_groups=9, bias=True)), (50, 512, 16, dict(score="sigmoid", groups=64, top_groups=8)),
          (37, 300, 64, dict(bias=True)), (6000, 16, 2, dict(bias=True))]


@pytest.mark.parametrize("tokens, experts, k, kw", ROUTES)
def test_route_experts(tokens, experts, k, kw):
    kw = dict(kw)
    logits = rand((tokens, experts), tokens, 1.5)
    bias = rand((experts,), 9, 0.1) if kw.pop("bias", False) else None
    r = routing().route_experts(logits.cuda(), k, bias=None if bias is None else bias.cuda(), **kw)
    ids, weights = O.route(logits, k, bias=bias, **kw)
    assert r.ids.tolist() == ids
    w = torch.tensor(weights, dtype=torch.float64)
    # expf, a sum of up to 512 terms over lanes and a quotient, twice: 64 u, and u |z - max| (at most 14 here) of the exponent's argument
    assert ((r.weights.cpu().double() - w).abs() <= 128 * U * w).all()
    check_order(r)


def test_route_experts_settles_what_fp32_does_not():
    """Biases that bring every key of a token to within an fp32 rounding of one another: fp64 decides, in groups too."""
    e = routing()
    logits = rand((24, 64), 1, 2.0)
    bias = (0.75 - torch.sigmoid(logits[:1].double())).float()[0]
    logits[1::2] = logits[0]
    logits[1::4] += torch.randint(-1, 2, (6, 64), generator=torch.Generator().manual_seed(2)) * 2.0 ** -22
    for kw in (dict(), dict(groups=8, top_groups=3), dict(groups=16, top_groups=5)):
        r = e.route_experts(logits.cuda(), 6, score="sigmoid", bias=bias.cuda(), **kw)
        assert r.ids.tolist() == O.route(logits, 6, "sigmoid", bias, **kw)[0]
    soft = torch.softmax(logits[0].double(), 0)
    bias = (0.5 - soft).float()
    r = e.route_experts(logits.cuda(), 6, bias=bias.cuda())
    assert r.ids.tolist() == O.route(logits, 6, "softmax", bias)[0]


def test_route_experts_equal_keys_take_the_lower_index():
    e = routing()
    r = e.route_experts(torch.zeros(3, 40, device="cuda"), 5)
    assert r.ids.tolist() == [[0, 1, 2, 3, 4]] * 3
    assert torch.allclose(r.weights, torch.full((3, 5), 0.2, device="cuda"))
    r = e.route_experts(torch.zeros(2, 40, device="cuda"), 3, score="sigmoid", groups=8, top_groups=2, bias=torch.zeros(40, device="cuda"))
    assert r.ids.tolist() == [[0, 1, 2]] * 2
    check_order(r)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kw", [{}, dict(bias=True), dict(bias=True, groups=4, top_groups=2)])
def test_route_experts_masked_and_broken_logits(score, kw):
    kw = dict(kw)
    x = rand((7, 16), 3)
    x[0] = -math.inf                                         # nothing left
    x[1, 3:] = -math.inf
    x[2, 5] = math.inf
    x[3] = math.nan
    x[4, ::2] = math.nan
    x[5] = torch.finfo(torch.float32).min
    bias = rand((16,), 4, 0.1) if kw.pop("bias", False) else None
    r = routing().route_experts(x.cuda(), 4, score=score, bias=None if bias is None else bias.cuda(), **kw)
    ids, weights = O.route(x, 4, score, bias, **kw)
    assert r.ids.tolist() == ids
    w = torch.tensor(weights, dtype=torch.float64)
    assert ((r.weights.cpu().double() - w).abs() <= 128 * U * w + 1e-37).all()
    check_order(r)


def test_route_experts_with_experts_that_a_bias_rules_out():
    x, bias = rand((20, 12), 1), torch.zeros(12)
    bias[2:] = -math.inf
    r = routing().route_experts(x.cuda(), 3, bias=bias.cuda())
    assert r.ids.tolist() == O.route(x, 3, bias=bias)[0] and all(set(i[:2]) == {0, 1} for i in r.ids.tolist())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top_groups, k", [(8, 3, 5), (4, 2, 9), (16, 7, 6)])
def test_route_experts_with_groups_that_a_bias_rules_out_or_forces(score, groups, top_groups, k):
    x, bias = rand((40, 64), 6), rand((64,), 7, 0.1)
    size = 64 // groups
    bias[size:3 * size] = -math.inf                          # two whole groups, and one but for a single expert
    bias[3 * size + 1:4 * size] = -math.inf
    r = routing().route_experts(x.cuda(), k, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups)
    assert r.ids.tolist() == O.route(x, k, score, bias, groups, top_groups)[0]
    bias[:] = -math.inf                                      # none but two experts of different groups are left
    bias[5], bias[60] = 0.0, 0.5
    r = routing().route_experts(x.cuda(), k, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups)
    assert r.ids.tolist() == O.route(x, k, score, bias, groups, top_groups)[0]
    bias[60] = math.inf
    r = routing().route_experts(x.cuda(), 1, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups)
    assert r.ids.flatten().tolist() == [60] * 40
    check_order(r)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts, groups, top_groups, k", [(16, 4, 1, 4), (32, 4, 2, 12), (64, 8, 2, 16), (12, 4, 2, 6), (200, 10, 2, 40), (128, 64, 3, 5)])
def test_route_experts_stays_in_the_best_groups_where_a_bias_rules_out_their_experts(score, experts, groups, top_groups, k):
    """A kept group with one finite key, the rest at -inf: those, and none of the groups that go, fill up the choice."""
    size = experts // groups
    x, bias = rand((20, experts), 8), torch.zeros(experts)
    for g in range(groups - top_groups, groups):
        bias[g * size:(g + 1) * size] = -math.inf
        bias[g * size] = bias[g * size + 1] = 5.0
    for b in (bias, torch.where(bias == 5.0, torch.tensor(math.inf), bias)):
        r = routing().route_experts(x.cuda(), k, score=score, bias=b.cuda(), groups=groups, top_groups=top_groups)
        assert all(e // size >= groups - top_groups for row in r.ids.tolist() for e in row)
        assert r.ids.tolist() == O.route(x, k, score, b, groups, top_groups)[0]
        check_order(r)
    b = bias.clone()                                         # an infinity beside -inf makes its group the best
    b[:size] = -math.inf
    b[0] = math.inf
    r = routing().route_experts(x.cuda(), k, score=score, bias=b.cuda(), groups=groups, top_groups=top_groups)
    assert r.ids.tolist() == O.route(x, k, score, b, groups, top_groups)[0]


def test_route_experts_takes_strided_and_16_bit_logits():
    x = rand((50, 40), 2)
    r = routing().route_experts(x.cuda()[:, 4:36], 3)
    assert r.ids.tolist() == O.route(x[:, 4:36], 3)[0]
    h = x.bfloat16()
    assert routing().route_experts(h.cuda(), 3).ids.tolist() == O.route(h.float(), 3)[0]
    assert routing().route_experts(x.t().contiguous().t().cuda(), 3).ids.tolist() == O.route(x, 3)[0]
    empty = routing().route_experts(torch.empty(0, 8, device="cuda"), 2)
    assert empty.ids.shape == (0, 2) and empty.starts.tolist() == [0] * 9


def test_route_experts_of_many_tokens_keeps_the_order():
    """Several chunks, uneven experts: against a stable sort."""
    x = rand((20000, 24), 5) + torch.linspace(0, 4, 24)
    r = routing().route_experts(x.cuda(), 3)
    ids = x.sort(dim=1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(r.ids.cpu().long(), ids)
    flat = ids.flatten()
    assert torch.equal(r.order.cpu().long(), flat.sort(stable=True).indices)
    assert torch.equal(r.place.cpu().long()[r.order.cpu().long()], torch.arange(60000))
    assert r.starts.tolist() == [int((flat < e).sum()) for e in range(25)]


# tokens, experts, k, width, ff
MLPS = [(1, 1, 1, 16, 16), (1, 8, 2, 256, 128), (5, 6, 2, 200, 150), (40, 3, 1, 128, 260), (64, 5, 3, 130, 96), (17, 12, 4, 520, 72), (300, 4, 2, 96, 128), (150, 2, 2, 384, 200)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens, n, k, width, ff", MLPS)
def test_expert_mlp(tokens, n, k, width, ff, dtype):
    e, f = routing(), ops()
    h = loud(tokens, width, tokens, torch.bfloat16)
    x = f.quantize_rows(h.cuda())
    w_in, in_wide = weight8((n, 2, ff, width), 1)
    w_out, out_wide = weight8((n, width, ff), 2)
    routes = e.route_experts(rand((tokens, n), 3).cuda(), k, score="sigmoid")
    add = rand((tokens, width), 4, dtype=dtype)
    for plus in (None, add):
        y = e.expert_mlp(x, w_in, w_out, routes, add=None if plus is None else plus.cuda(), dtype=dtype)
        err = product_error(max(width, ff))
        want, off, most = O.expert_mlp(O.wide_rows(*O.quantize(h.double())), [in_wide[2 * i:2 * i + 2] for i in range(n)], out_wide, routes.ids.tolist(),
                                       routes.weights.double().tolist(), err)
        if plus is not None:
            want, most = want + plus.double(), most + plus.double().abs()
        half = torch.finfo(dtype).eps / 2                    # an expert's result and the sum; k + 1 additions in fp32
        off = off + (2 * half + (k + 2) * U) * (most + off)
        assert y.dtype == dtype and ((y.cpu().double() - want).abs() <= off + 1e-40).all()


@pytest.mark.parametrize("tokens, n, k, width, ff", [(90, 5, 2, 264, 136), (100, 4, 2, 256, 300), (140, 4, 2, 136, 128), (33, 2, 2, 1032, 96)])
def test_expert_mlp_on_both_sides_of_the_choice_of_kernels(tokens, n, k, width, ff):
    """36, 50, 70 and 33 rows an expert."""
    test_expert_mlp(tokens, n, k, width, ff, torch.bfloat16)


@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_expert_mlp_rounds_small_sums_once(tokens):
    """What is summed is fp32 for either result: the 16-bit one is the other, rounded."""
    e, f = routing(), ops()
    w_in, w_out = weight8((8, 2, 128, 256), 1)[0], weight8((8, 256, 128), 2)[0]
    x = f.quantize_rows(rand((tokens, 256), 1, dtype=torch.bfloat16).cuda())
    routes = e.route_experts(rand((tokens, 8), 3).cuda(), 8)
    fine = e.expert_mlp(x, w_in, w_out, routes, dtype=torch.float32)
    assert torch.equal(e.expert_mlp(x, w_in, w_out, routes), fine.bfloat16())


def test_expert_mlp_of_more_results_than_are_kept_in_32_bits():
    """34 MB of them in fp32.  With one expert a token, whose weight is 1, rounding twice is rounding once."""
    e, f = routing(), ops()
    w_in, w_out = weight8((8, 2, 128, 256), 1)[0], weight8((8, 256, 128), 2)[0]
    x = f.quantize_rows(rand((33000, 256), 1, dtype=torch.bfloat16).cuda())
    routes = e.route_experts(rand((33000, 8), 3).cuda(), 1)
    assert (routes.weights == 1).all()
    fine = e.expert_mlp(x, w_in, w_out, routes, dtype=torch.float32)
    assert torch.equal(e.expert_mlp(x, w_in, w_out, routes), fine.bfloat16())


def test_expert_mlp_where_all_tokens_go_to_one_expert_and_others_have_none():
    e, f = routing(), ops()
    logits = torch.zeros(260, 9)
    logits[:, 4] = 5
    logits[::3, 7] = 3
    h = rand((260, 144), 1, dtype=torch.bfloat16)
    w_in, in_wide = weight8((9, 2, 136, 144), 1)
    w_out, out_wide = weight8((9, 144, 136), 2)
    routes = e.route_experts(logits.cuda(), 1)
    assert routes.starts.tolist() == [0] * 5 + [260] * 5
    y = e.expert_mlp(f.quantize_rows(h.cuda()), w_in, w_out, routes, dtype=torch.float32)
    want, off, most = O.expert_mlp(O.wide_rows(*O.quantize(h.double())), [in_wide[2 * i:2 * i + 2] for i in range(9)], out_wide, routes.ids.tolist(),
                                   routes.weights.double().tolist(), product_error(144))
    assert ((y.cpu().double() - want).abs() <= off + 4 * U * (most + off)).all()


def test_expert_mlp_a_broken_token_stays_by_itself_and_the_order_of_tokens_does_not_matter():
    e, f = routing(), ops()
    h = rand((90, 256), 1, dtype=torch.bfloat16)
    logits = rand((90, 6), 2)
    w_in, _ = weight8((6, 2, 128, 256), 3)
    w_out, _ = weight8((6, 256, 128), 4)

    def run(h, logits):
        return e.expert_mlp(f.quantize_rows(h.cuda()), w_in, w_out, e.route_experts(logits.cuda(), 2))

    a = run(h, logits)
    bad = h.clone()
    bad[17, 100], bad[40, 3] = math.nan, math.inf
    b = run(bad, logits)
    rest = [i for i in range(90) if i not in (17, 40)]
    assert torch.isnan(b[[17, 40]]).all() and torch.equal(a[rest], b[rest])
    p = torch.randperm(90, generator=torch.Generator().manual_seed(5))
    assert torch.equal(run(h[p], logits[p]), a[p.cuda()])
    assert torch.equal(run(h, logits), a)
    assert run(h[:0], logits[:0]).shape == (0, 256)


def test_expert_mlp_of_no_tokens_and_with_other_weights():
    e, f = routing(), ops()
    w_in, w_out = f.Fp8Weight.of(rand((4, 2, 64, 96), 1).cuda()), f.Fp8Weight.of(rand((4, 96, 64), 2).cuda())
    x = f.quantize_rows(rand((6, 96), 3).cuda())
    assert e.expert_mlp(x[:0], w_in, w_out, e.route_experts(torch.empty(0, 4, device="cuda"), 2)).shape == (0, 96)
    r = e.route_experts(rand((6, 4), 4).cuda(), 2)
    whole = e.expert_mlp(x, w_in, w_out, r, dtype=torch.float32)
    r.weights = 2 * r.weights                                # exact: so is the doubled sum
    assert torch.equal(e.expert_mlp(x, w_in, w_out, r, dtype=torch.float32), 2 * whole)


def test_operators_behind_copies_and_joined_streams_in_a_graph():
    """What stands in front of a launch that may begin early is a memset, a copy or another stream's kernel."""
    from atma_b200.decoder_ops import linear
    f = ops()
    src, w = rand((40, 256), 1).cuda(), f.Fp8Weight.of(rand((128, 256), 2).cuda())
    a, b = torch.empty_like(src), torch.empty_like(src)
    out = torch.empty(40, 128, device="cuda")

    def run(side):
        here = torch.cuda.current_stream()
        a.zero_()
        qa = f.quantize_rows(a)
        b.copy_(src)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b.mul_(0.5)
            qb = f.quantize_rows(b)
        a.copy_(src)
        here.wait_stream(side)
        f.linear_fp8(qb, w, out=out)
        return out + f.linear_fp8(qa, w, dtype=torch.float32) + linear(f.quantize_rows(a), w).float()

    side = torch.cuda.Stream()
    run(side)
    torch.cuda.synchronize()
    expected = run(side).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = run(side)
    for i in range(3):
        src.mul_(2.0)                                        # scales double, values stay
        result.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(result, expected * 2.0 ** (i + 1))


def test_norm_routing_and_experts_in_a_graph():
    """The layer's run of operators, captured: replays on other inputs do what the calls do."""
    e, f = routing(), ops()
    w_in, _ = weight8((8, 2, 64, 160), 1)
    w_out, _ = weight8((8, 160, 64), 2)
    weight, router = rand((160,), 3, 0.1, torch.bfloat16).cuda(), rand((8, 160), 4, 0.2).cuda()
    x, y = rand((12, 160), 5).cuda(), rand((12, 160), 6, dtype=torch.bfloat16).cuda()

    def layer(x, y, total):
        (rows, h), = f.residual_norms_fp8(x, y, [weight], 1e-6, out=total, plain=True)
        routes = e.route_experts(h.float() @ router.t(), 2)
        return e.expert_mlp(rows, w_in, w_out, routes, add=y)

    sx, sy, total = x.clone(), y.clone(), torch.empty_like(x)
    want = layer(x, y, total).clone(), total.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(sx, sy, total)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(sx, sy, total)
    sx.normal_(), sy.normal_()
    graph.replay()
    other = layer(sx, sy, torch.empty_like(x))
    torch.cuda.synchronize()
    assert torch.equal(out, other)
    sx.copy_(x), sy.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(total, want[1])


def test_expert_mlp_rounds_large_sums_once():
    """As many tokens as there may be: what is summed, here 35 MB of it, is fp32 for a 16-bit result too."""
    e, f = routing(), ops()
    w_in, w_out = weight8((4, 2, 128, 256), 1)[0], weight8((4, 256, 128), 2)[0]
    x = f.quantize_rows(rand((17000, 256), 1, dtype=torch.bfloat16).cuda())
    routes = e.route_experts(rand((17000, 4), 3).cuda(), 2)
    fine = e.expert_mlp(x, w_in, w_out, routes, dtype=torch.float32)
    assert torch.equal(e.expert_mlp(x, w_in, w_out, routes), fine.bfloat16())


def test_route_experts_groups_whose_keys_cancel_by_hand():
    """Sums of 0.980572 and 0.980638 of keys around 1e5 and -1e5: fp32 ones are 0.984375 and 0.9765625."""
    x, bias = torch.tensor([[0.07926305, -0.15725687, -0.8928827, 0.80069155]]), torch.tensor([1e5, -1e5, 1e5, -1e5])
    r = routing().route_experts(x.cuda(), 2, score="sigmoid", bias=bias.cuda(), groups=2, top_groups=1)
    assert r.ids.tolist() == O.route(x, 2, "sigmoid", bias, 2, 1)[0] == [[2, 3]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("most", [16.0, 64.0, 1e3, 1e4, 1e5, 1e6, 3e38])
@pytest.mark.parametrize("experts, groups, top_groups, k", [(4, 2, 1, 2), (64, 8, 3, 4), (24, 8, 3, 4), (160, 8, 3, 6), (128, 64, 7, 9)])
def test_route_experts_groups_whose_keys_cancel(experts, groups, top_groups, k, most, score):
    """The two best keys of every group are near a bias and near its opposite: their sum says nothing of what they are off by."""
    size = experts // groups
    bias = torch.full((groups, size), -1.125 * most if most < 1e38 else -math.inf)
    bias[:, 0], bias[:, 1] = most, -most
    x, bias = rand((600, experts), 11), bias.flatten()
    r = routing().route_experts(x.cuda(), k, score=score, bias=bias.cuda(), groups=groups, top_groups=top_groups)
    assert r.ids.tolist() == O.route(x, k, score, bias, groups, top_groups)[0]


# experts, k, options: lanes with one and with several experts, groups of no whole lanes, more choices than lanes
SMALL_SCORES = [(4, 2, {}), (64, 2, {}), (64, 7, dict(groups=8, top_groups=6)), (64, 40, {}), (24, 7, dict(groups=8, top_groups=7)), (300, 2, {}), (300, 40, {})]


def check_weights(r, logits, k, score, bias=None, **kw):
    """128 u as above, u |z - max| of the exponent's argument in a score and in the sum; what fp32 has no bits for."""
    ids, weights = O.route(logits, k, score, bias, **kw)
    assert r.ids.tolist() == ids
    w = torch.tensor(weights, dtype=torch.float64)
    span = float(logits.max() - logits.min()) if score == "softmax" else 0
    assert ((r.weights.cpu().double() - w).abs() <= (128 + 2 * span) * U * w + 2.0 ** -129).all()
    return w


@pytest.mark.parametrize("experts, k, kw", SMALL_SCORES)
@pytest.mark.parametrize("low, high", [(-98, -95), (-90, -80), (-105, -87), (-300, -90), (-120, -20), (-120, 3)])
def test_route_experts_weights_of_sigmoids_that_fp32_does_not_hold(experts, k, kw, low, high):
    x = low + (high - low) * torch.rand(60, experts, generator=torch.Generator().manual_seed(1))
    r = routing().route_experts(x.cuda(), k, score="sigmoid", **kw)
    w = check_weights(r, x, k, "sigmoid", **kw)
    assert ((w.sum(1) - 1).abs() < 1e-12).all()
    check_weights(routing().route_experts(x.cuda(), k, score="sigmoid", renormalize=False, **kw), x, k, "sigmoid", renormalize=False, **kw)


@pytest.mark.parametrize("experts, k, kw", SMALL_SCORES)
@pytest.mark.parametrize("gap", [60, 85, 95, 110, 200, 600])
def test_route_experts_weights_beside_a_larger_logit_that_is_kept_out(experts, k, kw, gap):
    x, bias = 3 * rand((60, experts), 5), torch.zeros(experts)
    x[:, 1] = gap
    bias[1] = -math.inf
    check_weights(routing().route_experts(x.cuda(), k, bias=bias.cuda(), **kw), x, k, "softmax", bias, **kw)
    if "groups" in kw:                                       # by its group
        bias = torch.zeros(experts)
        bias[:experts // kw["groups"]] = -3.0
        check_weights(routing().route_experts(x.cuda(), k, bias=bias.cuda(), **kw), x, k, "softmax", bias, **kw)


@pytest.mark.parametrize("tokens, n, k, width, ff, skew", [
    (64, 64, 2, 128, 1024, 0),       # 2 rows an expert, 16 tokens wide: 500 gated tiles for 296 CTAs
    (600, 48, 2, 130, 1024, 0),      # 25 rows, 32 wide: over 400
    (480, 24, 2, 128, 1100, 0),      # 40 rows, 64 wide, a CTA an SM: 220 and more
    (760, 24, 2, 128, 1300, 0),      # 63 rows, pairs of SMs: 264 tiles for 74
    (2400, 3, 1, 130, 2900, 9),      # ten tiles of one expert's rows, which go in bands of eight; the other experts have none
])
def test_expert_mlp_where_ctas_take_several_tiles(tokens, n, k, width, ff, skew):
    e, f = routing(), ops()
    h = loud(tokens, width, tokens, torch.bfloat16)
    w_in, in_wide = weight8((n, 2, ff, width), 1)
    w_out, out_wide = weight8((n, width, ff), 2)
    logits = rand((tokens, n), 3)
    logits[:, 0] += skew
    routes = e.route_experts(logits.cuda(), k, score="sigmoid")
    y = e.expert_mlp(f.quantize_rows(h.cuda()), w_in, w_out, routes, dtype=torch.float32)
    want, off, most = O.expert_mlp(O.wide_rows(*O.quantize(h.double())), [in_wide[2 * i:2 * i + 2] for i in range(n)], out_wide, routes.ids.tolist(),
                                   routes.weights.double().tolist(), product_error(max(width, ff)))
    off = off + (k + 4) * U * (most + off)                   # as in test_expert_mlp
    assert ((y.cpu().double() - want).abs() <= off + 1e-40).all()
    assert off.norm() < 0.03 * want.norm()                   # a tile in another's place would be off by all of it


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens, k, D", [(1, 1, 1), (5, 3, 20), (40, 8, 264), (7, 11, 1001)])
def test_weighted_sum_by_its_c_entry(tokens, k, D, dtype):
    """atma_combine_experts, for a caller with results of its own: k fmas in fp32 and one rounding."""
    from atma_b200 import _lib
    y, add, w = rand((tokens * k, D), 1, dtype=dtype), rand((tokens, D), 2, dtype=dtype), rand((tokens, k), 3)
    place = torch.randperm(tokens * k, generator=torch.Generator().manual_seed(4)).int()
    for plus in (None, add):
        on = [t if t is None else t.cuda() for t in (y, place, w, plus)]
        out = torch.full((tokens + 1, D), 7.0, device="cuda", dtype=dtype)
        rc = _lib.load_decoder().atma_combine_experts(*(None if t is None else t.data_ptr() for t in on), out.data_ptr(), tokens, k, D, _lib.DTYPE_CODE[dtype],
                                                      torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and (out[tokens] == 7).all()
        terms = y.double()[place.long()].view(tokens, k, D) * w.double()[..., None]
        want = terms.sum(1) + (0 if plus is None else plus.double())
        off = k * U * (terms.abs().sum(1) + (0 if plus is None else plus.double().abs()))
        off = off + (torch.finfo(dtype).eps / 2 * (want.abs() + off) if dtype is torch.bfloat16 else 0)
        assert ((out[:tokens].cpu().double() - want).abs() <= off).all()
