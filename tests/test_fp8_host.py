"""CPU: the oracle of the operators in 8 bits against itself, weights in 8 bits, and what the operators refuse."""

import ctypes
import math
import os
import subprocess
import tempfile
import textwrap

import pytest
import torch

from oracle import fp8 as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_e4m3_table_and_rounding():
    v = O.e4m3_values()
    assert len(v) == 127 and v[-1] == 448 and torch.equal(v.to(torch.float8_e4m3fn).double(), v)
    x = torch.cat([torch.linspace(-448, 448, 9973, dtype=torch.float64), v, -v])
    same = O.to_e4m3(x) == x.float().to(torch.float8_e4m3fn).double()
    assert same.all()
    b = O.borders()
    assert torch.equal(O.to_e4m3(b), b.float().to(torch.float8_e4m3fn).double())
    eps = 2.0 ** -40
    assert (O.to_e4m3(b * (1 + eps)) > O.to_e4m3(b * (1 - eps))).all()


@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (128, 128), (200, 300), (3, 130, 129), (2, 2, 64, 40)])
def test_weights_in_8_bits(shape):
    from atma_b200.fp8_ops import Fp8Weight
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    w8 = Fp8Weight.of(w)
    assert w8.shape == shape and w8.values.data_ptr() % 16 == 0 and (w8.values.stride(-2) % 16 == 0 or shape[:-1] == (1,))
    s = w8.scales.reshape(-1, *w8.scales.shape[-2:]).double()
    for m, q, sc in zip(w.reshape(-1, *shape[-2:]).double(), w8.values.reshape(-1, *shape[-2:]), s):
        for i in range(sc.shape[0]):
            for j in range(sc.shape[1]):
                at = (slice(i * 128, (i + 1) * 128), slice(j * 128, (j + 1) * 128))
                assert sc[i, j] == (m[at].abs().max() / 448).float()
                assert torch.equal(q[at].double(), O.to_e4m3(m[at] / sc[i, j]))
    assert (w8.wide() - w).abs().max() <= w.abs().max() * 2.0 ** -4
    assert torch.equal(Fp8Weight.of(torch.zeros(3, 4)).wide(), torch.zeros(3, 4))


def test_rows_and_weights_refuse_what_does_not_fit():
    from atma_b200.fp8_ops import E4M3, Fp8Rows, Fp8Weight
    v = torch.zeros(4, 256, dtype=E4M3)
    Fp8Rows(v, torch.zeros(4, 2))
    for values, scales in ((v.float(), torch.zeros(4, 2)), (v, torch.zeros(4, 1)), (v, torch.zeros(4, 2, dtype=torch.bfloat16)), (v[0], torch.zeros(2)),
                           (v, torch.zeros(2, 4))):
        with pytest.raises(ValueError):
            Fp8Rows(values, scales)
    for values, scales in ((v, torch.zeros(4, 2)), (v[0], torch.zeros(2)), (v.float(), torch.zeros(1, 2)), (v[None], torch.zeros(1, 2))):
        with pytest.raises(ValueError):
            Fp8Weight(values, scales)
    r = Fp8Rows(torch.zeros(4, 300, dtype=E4M3)[:, 3:260], torch.zeros(4, 3))            # odd addresses: copied
    assert r.values.data_ptr() % 16 == 0 and r.values.stride(0) % 16 == 0 and r.scales.stride() == (1, 4)
    w = Fp8Weight(torch.zeros(2, 300, 4, dtype=E4M3).transpose(1, 2), torch.zeros(2, 1, 3))
    assert w.values.stride() == (4 * 304, 304, 1)
    assert Fp8Rows(torch.zeros(1, 5, dtype=E4M3), torch.zeros(1, 1)).shape == (1, 5)


def test_operators_refuse_cpu_tensors():
    from atma_b200 import experts, fp8_ops as f
    x = torch.zeros(2, 128)
    r, w = f.Fp8Rows(torch.zeros(2, 128, dtype=f.E4M3), torch.zeros(2, 1)), f.Fp8Weight.of(torch.zeros(3, 128))
    calls = [lambda: f.quantize_rows(x), lambda: f.residual_norms_fp8(x, None, [x[0]], 1e-6), lambda: f.linear_fp8(r, w), lambda: experts.route_experts(x, 2)]
    for call in calls:
        with pytest.raises(RuntimeError):
            call()


@pytest.fixture()
def anywhere(monkeypatch):
    """Checks of arguments without a GPU: tensors count as being where they should, and no launch is reached."""
    from atma_b200 import experts, fp8_ops

    def launch(*a, **kw):
        raise AssertionError("a refused call came through")

    for m in (fp8_ops, experts):
        monkeypatch.setattr(m, "_here", lambda *a: None)
        monkeypatch.setattr(m._lib, "load_decoder", launch)
    return fp8_ops, experts


def test_refused_arguments(anywhere):
    f, e = anywhere
    x, y, w = torch.zeros(4, 256), torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256, dtype=torch.bfloat16)
    r, m = f.Fp8Rows(torch.zeros(4, 256, dtype=f.E4M3), torch.zeros(4, 2)), f.Fp8Weight.of(torch.zeros(8, 256))
    stack = f.Fp8Weight.of(torch.zeros(6, 2, 32, 256)), f.Fp8Weight.of(torch.zeros(6, 256, 32))
    routes = e.Routes(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2), 6, torch.zeros(23, dtype=torch.int32))
    z = torch.zeros(4, 12)
    refused = [
        lambda: f.quantize_rows(x.half()), lambda: f.quantize_rows(x[0]), lambda: f.quantize_rows(x[:, :0]),
        lambda: f.residual_norms_fp8(x, y, [], 1e-6), lambda: f.residual_norms_fp8(x, y, [None], 1e-6), lambda: f.residual_norms_fp8(x, y, [w, w, w], 1e-6),
        lambda: f.residual_norms_fp8(x, x, [w], 1e-6), lambda: f.residual_norms_fp8(x, y[:2], [w], 1e-6), lambda: f.residual_norms_fp8(x, y, [w[:5]], 1e-6),
        lambda: f.residual_norms_fp8(x.double(), y, [w], 1e-6), lambda: f.residual_norms_fp8(x.t(), y, [w], 1e-6),
        lambda: f.residual_norms_fp8(x, y, [w], 1e-6, out=y), lambda: f.residual_norms_fp8(x, y, [w.half()], 1e-6),
        lambda: f.linear_fp8(x, m), lambda: f.linear_fp8(r, x), lambda: f.linear_fp8(r, stack[1]), lambda: f.linear_fp8(r, f.Fp8Weight.of(torch.zeros(8, 128))),
        lambda: f.linear_fp8(r, m, dtype=torch.float16), lambda: f.linear_fp8(r, m, out=torch.zeros(4, 9)),
        lambda: f.linear_fp8(r, m, out=torch.zeros(8, 4).t()), lambda: f.linear_fp8(r, m, out=torch.zeros(4, 8, dtype=torch.float64)),
        lambda: f.linear_fp8(r, m, out=torch.zeros(1, 8).expand(4, 8)),
        lambda: f.gelu_gated_linear_fp8(r, m), lambda: f.gelu_gated_linear_fp8(x, m), lambda: f.gelu_gated_linear_fp8(r, f.Fp8Weight.of(torch.zeros(3, 8, 256))),
        lambda: f.gelu_gated_linear_fp8(r, f.Fp8Weight.of(torch.zeros(2, 8, 255))),
        lambda: e.route_experts(z, 0), lambda: e.route_experts(z, 13), lambda: e.route_experts(z, 2, score="relu"), lambda: e.route_experts(z, 2, groups=5),
        lambda: e.route_experts(z, 2, groups=4, top_groups=5), lambda: e.route_experts(z, 4, groups=4, top_groups=1), lambda: e.route_experts(z, 2, bias=z),
        lambda: e.route_experts(z.int(), 2), lambda: e.route_experts(z[0], 2), lambda: e.route_experts(torch.zeros(2, 513), 2), lambda: e.route_experts(z[:, :0], 1),
        lambda: e.route_experts(torch.zeros(2, 200), 65), lambda: e.route_experts(torch.zeros(2, 130), 2, groups=65),
        lambda: e.expert_mlp(x, *stack, routes), lambda: e.expert_mlp(r[:2], *stack, routes), lambda: e.expert_mlp(r, stack[1], stack[0], routes),
        lambda: e.expert_mlp(r, *stack, routes, dtype=torch.float16), lambda: e.expert_mlp(r, *stack, routes, add=x),
        lambda: e.expert_mlp(r, *stack, None),
    ]
    # results over what is read
    big, gate = torch.zeros(4, 512), f.Fp8Weight.of(torch.zeros(2, 256, 256))
    memory = torch.zeros(8, 256, dtype=f.E4M3)
    over = f.Fp8Rows(memory[:4], torch.zeros(2, 4).t())
    refused += [
        lambda: f.residual_norms_fp8(big.view(-1)[:1024].view(4, 256), None, [w], 1e-6, out=big.view(-1)[256:1280].view(4, 256)),
        lambda: f.residual_norms_fp8(x, y, [w], 1e-6, out=torch.as_strided(y.view(torch.float32), (2, 256), (256, 1)).expand(2, 256)),
        lambda: f.gelu_gated_linear_fp8(over, gate, out=over), lambda: f.gelu_gated_linear_fp8(over, gate, out=f.Fp8Rows(memory[2:6], torch.zeros(2, 4).t())),
        lambda: f.gelu_gated_linear_fp8(over, gate, out=f.Fp8Rows(memory[4:], over.scales)), lambda: f.gelu_gated_linear_fp8(over, gate, out=over.columns(0, 128)),
        lambda: f.linear_fp8(over, m, out=memory.view(torch.bfloat16)[:4, :8]), lambda: f.quantize_rows(memory.view(torch.float32)[:4, :64], out=over.columns(0, 128)),
        lambda: f.quantize_rows(memory.view(torch.bfloat16).view(-1)[:1024].view(4, 256), out=over),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_routes_with_other_weights(anywhere):
    """A user may put weights of their own into the routes; what the kernels could not read is refused."""
    f, e = anywhere
    r, stack = f.Fp8Rows(torch.zeros(4, 256, dtype=f.E4M3), torch.zeros(4, 2)), (f.Fp8Weight.of(torch.zeros(6, 2, 32, 256)), f.Fp8Weight.of(torch.zeros(6, 256, 32)))
    w = torch.zeros(4, 2)
    for bad in (w.double(), w.bfloat16(), w[:, :1], w.t().contiguous().t(), w[:3], w[0]):
        routes = e.Routes(torch.zeros(4, 2, dtype=torch.int32), bad, 6, torch.zeros(23, dtype=torch.int32))
        with pytest.raises(ValueError, match="weights"):
            e.expert_mlp(r, *stack, routes)


def test_routes_with_other_choices_are_refused(anywhere):
    """Places go with the choices that they were made for: fewer, more or other ones would send rows behind the scratch memory."""
    f, e = anywhere
    r, stack = f.Fp8Rows(torch.zeros(4, 256, dtype=f.E4M3), torch.zeros(4, 2)), (f.Fp8Weight.of(torch.zeros(6, 2, 32, 256)), f.Fp8Weight.of(torch.zeros(6, 256, 32)))
    routes = lambda k, plan, tokens=4: e.Routes(torch.zeros(tokens, k, dtype=torch.int32), torch.zeros(tokens, k), 6, plan)
    two = torch.zeros(2 * 4 * 2 + 7, dtype=torch.int32)
    with pytest.raises(AssertionError, match="came through"):
        e.expert_mlp(r, *stack, routes(2, two))
    some = routes(2, two)
    some.ids, some.weights = some.ids[:, :1].contiguous(), some.weights[:, :1].contiguous()               # the best one alone
    for x, bad in ((r, some), (r, routes(3, two)), (r, routes(1, two)), (r, routes(2, two.long())), (r, routes(2, two[None])), (r, routes(2, two[:22])),
                   (r, routes(2, torch.zeros(46, dtype=torch.int32)[::2])), (r[:3], routes(2, two, 3))):
        with pytest.raises(ValueError, match="places"):
            e.expert_mlp(x, *stack, bad)


def test_results_into_rows_that_were_copied_are_refused(anywhere):
    """Every other row of wider rows: their values lie where they did, their scales do not, and would stay as they were."""
    f, _ = anywhere
    big, x = f.Fp8Rows(torch.zeros(8, 256, dtype=f.E4M3), torch.zeros(2, 8).t()), torch.zeros(4, 256)
    gate, r = f.Fp8Weight.of(torch.zeros(2, 256, 256)), f.Fp8Rows(torch.zeros(4, 256, dtype=f.E4M3), torch.zeros(2, 4).t())
    for out in (big[::2], f.Fp8Rows(torch.zeros(4, 256, dtype=f.E4M3), torch.zeros(4, 2)), f.Fp8Rows(torch.zeros(4, 257, dtype=f.E4M3)[:, 1:], torch.zeros(2, 4).t())):
        for call in (lambda: f.quantize_rows(x, out=out), lambda: f.gelu_gated_linear_fp8(r, gate, out=out)):
            with pytest.raises(ValueError, match="copied"):
                call()
    for out in (big[2:6], f.Fp8Rows(torch.zeros(9, 272, dtype=f.E4M3)[::2], torch.zeros(3, 5).t())[:4].columns(0, 256), f.empty_rows(4, 256, "cpu")):
        assert not out.copied
        with pytest.raises(AssertionError, match="came through"):
            f.quantize_rows(x, out=out)


def test_routing_refuses_what_fp32_would_round(anywhere):
    """Logits that differ in 64 bits alone would be equal, and the lower index would win: a choice is as in 64-bit arithmetic or refused."""
    _, e = anywhere
    z = torch.zeros(4, 12)
    for call in (lambda: e.route_experts(z.double(), 2), lambda: e.route_experts(z, 2, bias=z[0].double()), lambda: e.route_experts(z, 2, bias=z[0].long())):
        with pytest.raises(ValueError, match="float32"):
            call()
    for logits, bias in ((z, None), (z.bfloat16(), z[0].half()), (z.half(), z[0].bfloat16())):
        with pytest.raises(AssertionError, match="came through"):
            e.route_experts(logits, 2, bias=bias)


def test_linear_refuses_a_type_that_it_would_not_give():
    from atma_b200 import decoder_ops
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(3, 128, dtype=torch.bfloat16)
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(ValueError, match="bfloat16"):
            decoder_ops.linear(x, w, dtype=dtype)
    assert decoder_ops.linear(x, w, dtype=torch.bfloat16).dtype == decoder_ops.linear(x, w).dtype == torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    from atma_b200 import _lib
    if not os.path.exists(_lib.DECODER_LIB_PATH):
        from atma_b200.build import build
        build("decoder")
    return _lib.load_decoder()


def test_the_c_entries_refuse_before_they_launch(lib):
    from atma_b200 import _lib
    bad = _lib.ATMA_ERR_INVALID
    p = ctypes.c_void_p(4096)
    assert lib.atma_linear_fp8(None, None) == bad
    good = dict(x=4096, x_rs=256, x_scales=4096, xs_bs=4, w=4096, w_rs=256, w_scales=4096, out=4096, out_rs=64, M=4, N=64, K=250, groups=1, form=0, dtype=1)
    for change in (dict(dtype=2), dict(M=-1), dict(N=0), dict(K=0), dict(groups=0), dict(groups=3), dict(form=2), dict(N=63, form=1), dict(form=1), dict(groups=513, starts=4096), dict(x=0), dict(w=0),
                   dict(out=0), dict(x_scales=0), dict(w_scales=0), dict(x=4100), dict(w=4104), dict(x_rs=250), dict(w_rs=240), dict(x_rs=240), dict(out_rs=63),
                   dict(xs_bs=3), dict(M=1 << 30)):
        a = _lib.Fp8Args(**{**good, **change})
        assert lib.atma_linear_fp8(ctypes.byref(a), None) == bad, change
    assert lib.atma_linear_fp8(ctypes.byref(_lib.Fp8Args(**{**good, "M": 0})), None) == 0
    assert lib.atma_quantize_rows(p, 8, p, 8, p, 2, 2, 8, 2, None) == bad                # fp16
    assert lib.atma_quantize_rows(None, 8, p, 16, p, 2, 2, 8, 0, None) == bad
    assert lib.atma_quantize_rows(p, 8, p, 4, p, 2, 2, 8, 0, None) == bad
    assert lib.atma_quantize_rows(p, 8, p, 16, p, 1, 2, 8, 0, None) == bad
    assert lib.atma_quantize_rows(p, 8, p, 16, p, 1, 0, 8, 0, None) == 0
    route = lambda tokens=4, experts=8, k=2, groups=1, top=1, logits=p, starts=p, l_rs=8: lib.atma_route_experts(
        logits, l_rs, None, p, p, p, p, starts, p, tokens, experts, k, 0, groups, top, 1, 1.0, None)
    for kw in (dict(tokens=-1), dict(experts=0), dict(experts=513, l_rs=600), dict(k=0), dict(k=9), dict(groups=3), dict(groups=4, top=5), dict(groups=4, top=0),
               dict(k=3, groups=4), dict(logits=None), dict(starts=None), dict(l_rs=7), dict(tokens=1 << 30, k=2)):
        assert route(**kw) == bad, kw
    assert lib.atma_residual_norms_fp8(p, None, None, p, None, p, None, None, None, None, None, 2, 8, 16, 2, 1e-6, 1.0, 0, None) == bad
    assert lib.atma_combine_experts(p, p, p, None, None, 2, 2, 8, 0, None) == bad
    mlp = dict(x=4096, x_rs=16, x_scales=4096, xs_bs=2, w_gate_up=4096, w_gate_up_rs=16, w_gate_up_scales=4096, w_down=4096, w_down_rs=16, w_down_scales=4096,
               place=4096, starts=4096, weights=4096, out=4096, tokens=2, copies=2, experts=3, width=16, ff=16, dtype=1)
    assert lib.atma_expert_mlp(None, p, None) == bad
    for change in (dict(dtype=2), dict(tokens=-1), dict(copies=0), dict(width=0), dict(ff=0), dict(place=0), dict(starts=0), dict(weights=0), dict(out=0)):
        assert lib.atma_expert_mlp(ctypes.byref(_lib.ExpertArgs(**{**mlp, **change})), p, None) == bad, change
    assert lib.atma_expert_mlp(ctypes.byref(_lib.ExpertArgs(**mlp)), None, None) == bad
    assert lib.atma_expert_mlp(ctypes.byref(_lib.ExpertArgs(**mlp)), ctypes.c_void_p(4096 + 16), None) == bad
    assert lib.atma_expert_mlp(ctypes.byref(_lib.ExpertArgs(**{**mlp, "tokens": 0})), None, None) == 0
    assert lib.atma_expert_mlp_scratch_bytes(3, 2, 20, 130, 1) >= 6 * (32 + 4 + 144 + 8 + 40) and lib.atma_expert_mlp_scratch_bytes(0, 2, 20, 130, 1) == 0
    assert lib.atma_scatter_rows_fp8(p, 16, p, 2, p, 0, p, 16, p, 4, 2, 16, None) == bad


def test_argument_layouts_match_the_header():
    from atma_b200 import _lib
    src = '#include <stdio.h>\n#include "atma_decoder.h"\nint main(void) { printf("%zu %zu\\n", sizeof(atma_fp8_args), sizeof(atma_expert_args)); return 0; }\n'
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        open(c, "w").write(textwrap.dedent(src))
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        assert [ctypes.sizeof(_lib.Fp8Args), ctypes.sizeof(_lib.ExpertArgs)] == [int(n) for n in subprocess.check_output([exe]).split()]


def test_routing_oracle_by_hand():
    ids, w = O.route(torch.tensor([[1.0, 3.0, 2.0, 3.0]]), 2)
    assert ids == [[1, 3]] and w == [[0.5, 0.5]]
    z = torch.tensor([[0.0, 5.0, 1.0, 1.0, 4.0, -9.0]])
    ids, w = O.route(z, 2, "sigmoid", torch.tensor([0, -2.0, 0, 0, 0, 0]), 3, 1, renormalize=False)
    assert ids == [[2, 3]] and math.isclose(w[0][0], 1 / (1 + math.exp(-1)))
    assert O.order([[2, 0], [0, 1]], 4) == ([1, 2, 3, 0], [3, 0, 1, 2], [0, 2, 3, 4, 4])


def test_register_hand_over_of_the_pair_kernel_fits_the_launch():
    """The counts that setmaxnreg asks for add up to no more than the CTA is launched with; see the compiler's report of the build."""
    import re
    src = open(os.path.join(ROOT, "atma_b200", "csrc", "linear_fp8.cu")).read()
    log = os.path.join(ROOT, "atma_b200", "build", "linear_fp8.o.log")
    if not os.path.exists(log):
        pytest.skip("no compiler report (the library was not built in this tree)")
    dec, inc = (int(re.search(rf"setmaxnreg\.{w}\.sync\.aligned\.u32 (\d+);", src).group(1)) for w in ("dec", "inc"))
    used = [int(n) for n in re.findall(r"pair_kernel.*?Used (\d+) registers", open(log).read(), re.S)]
    assert len(used) == 3 and all(128 * dec + 256 * inc <= 384 * n for n in used), (dec, inc, used)
    # sums that do not stay in registers cost half of the rate (232 -> 360 us), and small changes decide whether they do
    assert re.findall(r"pair_kernel[^\n]*\n.*?(\d+) bytes spill stores", open(log).read(), re.S) == ["0"] * 3


# ---- models --------------------------------------------------------------------------------------------------------------
def test_oracle_of_layers_in_8_bits_is_near_the_plain_one():
    """Roundings to 8 bits are half a step of 2^-4 at most, evenly spread: a projection's result is off by 3.6 %, root mean square; of 32
    projections one behind another 20 %, as a root of the sum of squares."""
    from oracle import rizurax as R
    from tests.fp8_util import CONFIGS_8
    from tests.rizurax_util import logit_error
    cfg = CONFIGS_8["dense"]
    w, t = O.rizurax_weights(cfg, 7), list(range(30))
    a, b = O.rizurax_forward(cfg, w, t), R.forward(cfg, w, t)[0]
    e = logit_error(a, b)
    assert 1e-3 < e.median() and e.pow(2).mean().sqrt() < 0.2
    plain = {**cfg, "weights": None}
    assert torch.allclose(O.rizurax_forward(plain, w, t), b, rtol=1e-9, atol=1e-9)


def test_models_with_8_bits_and_experts_are_built_and_refused():
    from atma_b200.fp8_ops import Fp8Weight
    from atma_b200.rizurax import RizuraxModel
    from tests.fp8_util import CONFIGS_8, experts
    for name, cfg in CONFIGS_8.items():
        w = O.rizurax_weights(cfg, 7)
        m = RizuraxModel(cfg, w, torch.float32, "cpu")
        for layer, entry in zip(m.layers, cfg["layers"]):
            eight = cfg.get("weights") == "e4m3"
            assert isinstance(layer.w_out, Fp8Weight) == isinstance(layer.mixer.w_in, Fp8Weight) == eight
            if eight and layer.ff:
                assert layer.w_out.shape[1] == layer.mixed + layer.ff and layer.mixed % 128 == 0
                assert not layer.w_out.wide()[:, layer.mixer.width:layer.mixed].any()
            if layer.experts is not None:
                assert layer.experts.w_gate_up.shape[1] == 2 and layer.ff == 0
        assert m.weight_bytes() > 0 and m.new_state(2, 4, 16)
    cfg = CONFIGS_8["both"]
    with pytest.raises(ValueError, match="unknown weights"):
        RizuraxModel({**cfg, "weights": "int4"}, O.rizurax_weights(cfg, 7), torch.float32, "cpu")
    with pytest.raises(KeyError, match="router"):
        RizuraxModel(cfg, {n: t for n, t in O.rizurax_weights(cfg, 7).items() if not n.endswith("router")}, torch.float32, "cpu")
    bad = {**cfg, "layers": [experts(cfg["layers"][0], 15, 3, 128)] + cfg["layers"][1:]}
    with pytest.raises(ValueError, match="router"):
        RizuraxModel(bad, O.rizurax_weights(cfg, 7), torch.float32, "cpu")


def test_columns_of_rows_in_8_bits():
    from atma_b200.fp8_ops import E4M3, Fp8Rows
    r = Fp8Rows(torch.zeros(3, 400, dtype=E4M3), torch.zeros(3, 4))
    c = r.columns(128, 400)
    assert c.shape == (3, 272) and c.values.data_ptr() == r.values.data_ptr() + 128 and c.row_stride == r.row_stride
    assert c.scales.shape == (3, 3) and c.scales.data_ptr() == r.scales.data_ptr() + 4 * 3
    assert r.columns(0, 256, 200).shape == (3, 200)
    for a, b, used in ((64, 256, None), (0, 100, None), (0, 401, None), (128, 128, None), (0, 256, 100), (0, 256, 257)):
        with pytest.raises(ValueError):
            r.columns(a, b, used)
