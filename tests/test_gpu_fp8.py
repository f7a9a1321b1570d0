"""GPU: rows and weights in 8 bits - quantisation, the residual stream's norms, products - against fp64 (oracle/fp8.py).

What may be off, with u = 2^-24 (half a step of fp32):
  quantize_rows   nothing: scale and value are defined by one rounding each
  norms           the sum by u; a norm by 64 u: its sum of squares has at most 32 + 5 + 8 additions one behind another (half of that in the
                  root), six roundings follow.  A value of 8 bits moves over a border only where fp64's quotient is that near to one
  products        2 u for every addition inside of a block of 128 columns, whose partial sums its own |x| |w|^T bounds, then one addition for
                  every block, and three roundings of its scale: (2 * 128 + blocks + 3) u |x| |w|^T; 2^-8 more in bfloat16
"""

import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def ops():
    from atma_b200 import fp8_ops
    return fp8_ops


def rand(shape, seed, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def loud(rows, width, seed, dtype=torch.float32):
    """Rows with some channels far above the others and blocks of zeros and of tiny values."""
    x = rand((rows, width), seed)
    x[:, ::37] *= 30
    if width > 256 and rows > 1:
        x[1, 128:256] = 0
        x[0, 128:256] *= 1e-41
    return x.to(dtype)


def rows8(x):
    """Fp8Rows of an fp32 matrix by the oracle, and what they stand for."""
    q, s = O.quantize(x.double())
    f = ops()
    r = f.Fp8Rows(q.to(f.E4M3).cuda(), s.float().cuda())
    return r, O.wide_rows(q, s)


def weight8(shape, seed):
    f = ops()
    w = rand(shape, seed, shape[-1] ** -0.5)
    w8 = f.Fp8Weight.of(w)
    lead = w8.values.reshape(-1, *shape[-2:]), w8.scales.reshape(-1, *w8.scales.shape[-2:])
    return f.Fp8Weight(w8.values.cuda(), w8.scales.cuda()), [O.wide_weight(v, s) for v, s in zip(*lead)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, width", [(1, 1), (3, 5), (1, 128), (2, 127), (5, 129), (7, 516), (33, 1000), (64, 2048), (3, 8196), (2, 20001)])
def test_quantize_rows_is_the_definition(rows, width, dtype):
    x = loud(rows, width, rows * width, dtype)
    if width > 3:                                                        # borders: multiples of half steps of a scale that is a power of two
        n = min(width, 128)
        x[-1, :n] = torch.linspace(-448, 448, n).round().to(dtype)
        x[-1, 0] = 448
    r = ops().quantize_rows(x.cuda())
    q, s = O.quantize(x.double())
    assert torch.equal(r.scales.cpu().double(), s)
    assert torch.equal(r.values.cpu().double(), q)
    assert r.values.data_ptr() % 16 == 0 and (rows == 1 or r.values.stride(0) % 16 == 0 and r.scales.stride(0) == 1)


def test_quantize_rows_of_16_bit_values_over_borders():
    """16-bit values over a 16-bit largest one: exact quotients on borders and within 2^-25 of them, in every block."""
    x = torch.empty(256, 1024, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    x.copy_(torch.randint(-255, 256, x.shape, generator=g).float() / 16)
    x[:, ::128] = (7 * torch.randint(20, 36, (256, 8), generator=g)).float() / 8
    r = ops().quantize_rows(x.cuda())
    q, s = O.quantize(x.double())
    ties = torch.isin((x.double() / s.repeat_interleave(128, 1)).abs(), O.borders()).sum()
    assert ties > 1000
    assert torch.equal(r.values.cpu().double(), q) and torch.equal(r.scales.cpu().double(), s)


def test_quantize_rows_takes_strided_rows_and_odd_addresses():
    big = loud(9, 700, 3, torch.bfloat16).cuda()
    for x in (big[:, 4:516], big[:, 1:400], big[::2, :512], big.t()[:300].t(), big[:, 3:4]):
        a, b = ops().quantize_rows(x), ops().quantize_rows(x.contiguous())
        assert torch.equal(a.values.float(), b.values.float()) and torch.equal(a.scales, b.scales)


def test_a_row_with_nan_or_infinity_keeps_it_to_itself():
    f = ops()
    x = rand((4, 300), 1)
    x[1, 200], x[2, 5] = float("nan"), float("inf")
    r = f.quantize_rows(x.cuda())
    clean, _ = O.quantize(x[::3].double())
    assert torch.equal(r.values[::3].cpu().double(), clean)
    w, wide = weight8((40, 300), 2)
    y = f.linear_fp8(r, w, dtype=torch.float32).cpu()
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[::3]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, width, norms", [(1, 1, 1), (3, 100, 2), (2, 128, 1), (5, 130, 2), (4, 1000, 2), (9, 2048, 2), (1, 4097, 1), (3, 8192, 2),
                                                (2, 9000, 1), (300, 516, 2)])
def test_residual_norms_fp8(rows, width, norms, dtype):
    f = ops()
    x, y = loud(rows, width, 1), rand((rows, width), 2, dtype=dtype)
    ws = [rand((width,), 3 + i, 0.2, dtype) for i in range(norms)]
    total = torch.empty(rows, width, device="cuda")
    got = f.residual_norms_fp8(x.cuda(), y.cuda(), [w.cuda() for w in ws], 1e-6, out=total, plain=True)
    t = x.double() + y.double()
    assert ((total.cpu().double() - t).abs() <= U * t.abs() + 1e-45).all()
    for i, ((r, h), w) in enumerate(zip(got, ws)):
        want = O.norm(t, w.double(), 1e-6, 1.0)
        q, s = O.quantize(want)
        assert ((r.scales.cpu().double() - s).abs() <= 66 * U * s).all()
        ratio = want / s.repeat_interleave(128, 1)[:, :width]
        b = O.borders()
        near = (ratio.abs()[..., None] - b[torch.searchsorted(b, ratio.abs())[..., None].add(torch.tensor([-1, 0])).clamp(0, 125)]).abs().amin(-1) <= 132 * U * ratio.abs()
        mine = r.values.cpu().double()
        assert (near | (mine == q)).all() and ((mine - q).abs() <= 1.01 * O.step_at(ratio * 1.07)).all()
        assert near.float().mean() < 0.01 or width < 200
        if i == norms - 1:
            assert ((h.cpu().double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 64 * U) * want.abs()).all()
        else:
            assert h is None


def test_residual_norms_fp8_in_place_without_y_and_skipped():
    f = ops()
    x, w = rand((6, 640), 1).cuda(), rand((640,), 2, 0.1, torch.bfloat16).cuda()
    y = rand((6, 640), 3, dtype=torch.bfloat16).cuda()
    (a, _), = f.residual_norms_fp8(x, None, [w], 1e-5)
    kept = x.clone()
    none, (b, h) = f.residual_norms_fp8(x, None, [None, w], 1e-5, plain=True)
    assert none == (None, None) and torch.equal(x, kept) and torch.equal(a.values.float(), b.values.float()) and torch.equal(a.scales, b.scales)
    f.residual_norms_fp8(x, y, [w], 1e-5)
    assert torch.equal(x, kept + y.float())
    from atma_b200 import decoder_ops
    plain, = decoder_ops.residual_norms(x.clone(), None, (w,), 1e-5)
    (c, hc), = f.residual_norms_fp8(x, None, [w], 1e-5, plain=True)
    assert torch.equal(hc, plain)
    (d, _), = f.residual_norms_fp8(x, None, [w], 1e-5, offset=0.0)
    assert not torch.equal(c.scales, d.scales)


def product_error(K):
    return (2 * min(K, 128) + -(-K // 128) + 3) * U


def product_bound(x, w, dtype):
    want = x @ w.t()
    off = product_error(x.shape[1]) * (x.abs() @ w.abs().t())
    return want, off + (torch.finfo(dtype).eps / 2 * (want.abs() + off) if dtype != torch.float32 else 0)


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 3, 130), (1, 2048, 1024), (16, 300, 777), (17, 64, 128), (33, 129, 127), (64, 1000, 256), (65, 40, 2000), (127, 128, 384),
          (128, 256, 128), (129, 257, 144), (200, 513, 640), (255, 130, 1152), (257, 384, 512), (300, 1000, 1304), (513, 520, 260), (1000, 260, 900),
          (2600, 2000, 200), (40, 40000, 128),                            # more tiles than there are CTAs
          (3, 300000, 16), (130, 270000, 16)]                             # vocabularies: tiles of columns in thousands


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M, N, K", SHAPES)
def test_linear_fp8(M, N, K, dtype):
    x, xw = rows8(loud(M, K, 7 * M + K))
    w, ww = weight8((N, K), N)
    y = ops().linear_fp8(x, w, dtype=dtype)
    assert y.dtype == dtype and y.shape == (M, N)
    want, off = product_bound(xw, ww[0], dtype)
    assert ((y.cpu().double() - want).abs() <= off + 1e-40).all()


def test_linear_fp8_where_scales_differ_widely():
    """Blocks of one row and of one weight whose scales are 2^20 apart: every block is scaled by itself."""
    f = ops()
    x, _ = rows8(rand((70, 640), 1))
    w, _ = weight8((200, 640), 2)
    xs, ws = x.scales.clone(), w.scales.clone()
    xs *= torch.ldexp(torch.ones(5), torch.tensor([0, 20, -20, 10, 3])).cuda()
    ws *= torch.ldexp(torch.ones(5), torch.tensor([10, -20, 20, -10, 3])).cuda()
    x, w = f.Fp8Rows(x.values, xs), f.Fp8Weight(w.values, ws)
    want, off = product_bound(O.wide_rows(x.values.cpu(), xs.cpu()), O.wide_weight(w.values.cpu(), ws.cpu()), torch.float32)
    assert ((f.linear_fp8(x, w, dtype=torch.float32).cpu().double() - want).abs() <= off).all()


@pytest.mark.parametrize("M", [3, 150, 400])
def test_linear_fp8_takes_slices_copies_what_is_not_aligned_and_keeps_to_its_place(M):
    f = ops()
    x, xw = rows8(rand((M + 9, 520), 4))
    w, ww = weight8((300, 520), 5)
    want, off = product_bound(xw, ww[0], torch.bfloat16)
    assert ((f.linear_fp8(x[5:5 + M], w).cpu().double() - want[5:5 + M]).abs() <= off[5:5 + M]).all()
    odd = f.Fp8Rows(torch.empty(M + 9, 521, device="cuda", dtype=f.E4M3)[:, 1:].copy_(x.values), x.scales.contiguous())
    assert odd.values.data_ptr() % 16 == 0
    a, b = f.linear_fp8(odd, w), f.linear_fp8(x, w)
    assert torch.equal(a, b)
    wide = torch.full((M + 11, 700), 3.0, device="cuda", dtype=torch.bfloat16)
    for c0 in (8, 13):
        wide.fill_(3.0)
        f.linear_fp8(x, w, out=wide[1:M + 10, c0:c0 + 300])
        assert torch.equal(wide[1:M + 10, c0:c0 + 300], a)
        wide[1:M + 10, c0:c0 + 300] = 3.0
        assert (wide == 3.0).all()


def test_linear_fp8_of_no_rows():
    f = ops()
    w, _ = weight8((30, 64), 1)
    assert f.linear_fp8(f.quantize_rows(torch.empty(0, 64, device="cuda")), w).shape == (0, 30)


@pytest.mark.parametrize("M", [5, 300])
def test_products_in_a_graph_and_on_another_stream(M):
    f = ops()
    xin = rand((M, 384), 1, dtype=torch.bfloat16).cuda()
    w, _ = weight8((520, 384), 2)
    want = f.linear_fp8(f.quantize_rows(xin), w).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = f.linear_fp8(f.quantize_rows(xin), w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    static = xin.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f.linear_fp8(f.quantize_rows(static), w)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        also = f.linear_fp8(f.quantize_rows(static * 2), w)
    static.copy_(xin)
    graph.replay(), second.replay(), graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(also, want * 2)
    static.copy_(-xin)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, -want)


@pytest.mark.parametrize("M, N, K", [(1, 1, 16), (2, 130, 64), (16, 256, 512), (16, 128, 2048), (31, 200, 256), (64, 100, 1024), (100, 136, 300), (128, 384, 128),
                                     (129, 200, 256), (300, 264, 520), (520, 130, 1000)])
def test_gelu_gated_linear_fp8(M, N, K):
    f = ops()
    x, xw = rows8(rand((M, K), M))
    w, (gate, up) = weight8((2, N, K), N)
    r = f.gelu_gated_linear_fp8(x, w)
    assert r.shape == (M, N)
    err = product_error(K)
    g, u = xw @ gate.t(), xw @ up.t()
    eg, eu = err * (xw.abs() @ gate.abs().t()), err * (xw.abs() @ up.abs().t())
    a = O.gelu_tanh(g) * u
    ea = 1.13 * eg * (u.abs() + eu) + O.gelu_tanh(g).abs() * eu + 2e-5 * a.abs()
    q, s = O.quantize(a)
    es = torch.stack([ea[:, b * 128:(b + 1) * 128].amax(1) / 448 for b in range(s.shape[1])], 1) + U * s
    assert ((r.scales.cpu().double() - s).abs() <= es).all()
    wide = lambda t: t.repeat_interleave(128, 1)[:, :N]
    ratio = a / wide(s)
    off = (ea + ratio.abs() * wide(es)) / wide(s)
    mine = r.values.cpu().double()
    assert ((mine - ratio).abs() <= O.step_at(mine) / 2 * 1.0001 + off + O.step_at(ratio) * (off > 0) * 0.5).all()
    near = (O.to_e4m3(ratio - off) != O.to_e4m3(ratio + off))
    assert (near | (mine == q)).all()


@pytest.mark.parametrize("M, K", [(9, 512), (30, 300), (60, 512), (60, 2048), (120, 512), (300, 512)])
def test_a_row_does_not_depend_on_its_neighbours(M, K):
    """Rows in another order: each has the same bits."""
    f = ops()
    x, w, g = rand((M, K), M).cuda(), f.Fp8Weight.of(rand((200, K), 1, K ** -0.5).cuda()), f.Fp8Weight.of(rand((2, 1000, K), 2, 2 * K ** -0.5).cuda())
    p = torch.randperm(M, generator=torch.Generator().manual_seed(3)).cuda()
    a, b = f.quantize_rows(x), f.quantize_rows(x[p])
    assert torch.equal(f.linear_fp8(a, w, dtype=torch.float32)[p], f.linear_fp8(b, w, dtype=torch.float32))
    a, b = f.gelu_gated_linear_fp8(a, g), f.gelu_gated_linear_fp8(b, g)
    assert torch.equal(a.scales[p], b.scales) and torch.equal(a.values.view(torch.uint8)[p], b.values.view(torch.uint8))


@pytest.mark.parametrize("M, N, K", [(31, 300, 700), (32, 300, 700), (33, 130, 4224), (65, 520, 2560), (65, 520, 2688), (100, 19000, 200), (50, 9500, 136),
                                     (200, 130, 8192), (257, 256, 4104), (400, 128, 4096)])
def test_products_on_both_sides_of_the_choice_of_kernels(M, N, K):
    test_linear_fp8(M, N, K, torch.float32)
    test_gelu_gated_linear_fp8(M, N // 2, K)


def test_products_leave_no_status():
    """The bounded waits of the tensor-core kernels: none of this file's launches ran one out."""
    from atma_b200 import decoder_ops
    f = ops()
    x, _ = rows8(rand((300, 256), 1))
    w, _ = weight8((256, 256), 2)
    f.linear_fp8(x, w), f.linear_fp8(x[:7], w)
    assert decoder_ops.device_status() == 0


@pytest.mark.parametrize("M, N, K", [(4, 60000, 200), (20, 60000, 130), (600, 12000, 200)])
def test_gelu_gated_linear_fp8_where_ctas_take_several_tiles(M, N, K):
    """469 tiles for 296 CTAs, 16 and 32 tokens wide, and 282 for 74 pairs: barriers, largest values and scales of one tile after another."""
    test_gelu_gated_linear_fp8(M, N, K)


def test_a_row_alone_is_as_near_as_in_a_batch():
    """Other numbers of rows take other kernels and orders of sums: the last bits may differ, the bound holds for each."""
    f = ops()
    x, xw = rows8(rand((300, 2048), 4))
    w, ww = weight8((520, 2048), 5)
    want, off = product_bound(xw, ww[0], torch.float32)
    for n in (1, 7, 20, 50, 130, 300):
        assert ((f.linear_fp8(x[:n], w, dtype=torch.float32).cpu().double() - want[:n]).abs() <= off[:n]).all()
