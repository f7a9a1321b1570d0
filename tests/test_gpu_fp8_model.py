"""GPU: Rizurax with its projections in 8 bits and with experts, through the engine, against fp64 (oracle/fp8.py).

In float32 the two sides differ as any float32 run does (a few 1e-6) until that moves a value of 8 bits over a border, once in some
30 000 values (2e-6 of a step of 2^-4 on either side); such a value is off by a step, 2^-3 of itself at most, one of 64 or more in
a sum: 1.6 % of a projection's result, in its token and, less, in all later ones, which see its keys and its state.  A token has up to
3000 values, so that the tokens in front of the first such one are some ten, or few: they have to be as near as float32
runs are (tests/test_gpu_rizurax.py: 1.2e-4), at least one of them, and all tokens within four such values: 6.4 %.
In bfloat16 every value is off by up to 2^-9 before it is rounded to 8 bits, and results differ as roundings do: a half step of 2^-4
evenly spread is 3.6 % of a projection's result, in up to four projections of up to eight layer runs one behind another: 20 % (as a
root of the sum of squares, 3.6 % * sqrt(32)).  That is a root mean square; a token's own result has no such bound, least of all where
2^-9 of a router's logits (of 64 to 128 products each) chooses another of two experts as near, whose feed-forward is another altogether.
With keys of a spread of 1 in 2^-9 sqrt(2) of each other, that is one choice in some 100, three of them a layer: so nine tokens of ten.
"""

import json

import pytest
import torch

from oracle import fp8 as O
from tests.fp8_util import CONFIGS_8
from tests.rizurax_util import logit_error, prompt

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
_models, _wanted = {}, {}


def model(name, dtype):
    if (name, dtype) not in _models:
        from atma_b200.rizurax import RizuraxModel
        cfg = CONFIGS_8[name]
        _models[name, dtype] = cfg, RizuraxModel(cfg, O.rizurax_weights(cfg, 7), dtype)
    return _models[name, dtype]


def wanted(name, tokens):
    key = name, tuple(tokens)
    if key not in _wanted:
        _wanted[key] = O.rizurax_forward(CONFIGS_8[name], O.rizurax_weights(CONFIGS_8[name], 7), tokens)
    return _wanted[key]


def engine(m, **kw):
    from atma_b200.engine import Engine
    return Engine(m, **{"max_tokens": 1200, "max_seqs": 6, "block_size": 128, **kw})


def close(got, want, dtype):
    e = logit_error(got, want)
    if dtype == F32:
        assert e.max() < 0.064 and e.min() < 1.2e-4, e.tolist()
    else:
        assert e.sort().values[int(0.9 * (len(e) - 1))] < 0.2, e.tolist()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", list(CONFIGS_8))
@pytest.mark.parametrize("cuts", [(40,), (1,) * 20, (17, 1, 1, 9, 2)])
def test_prompts_portions_and_single_tokens(name, dtype, cuts):
    cfg, m = model(name, dtype)
    t = prompt(sum(cuts), cfg["vocab"], len(cuts))
    e, got, at = engine(m), [], 0
    for n in cuts:
        got.append(e.feed([("a", t[at:at + n], list(range(n)))]))
        at += n
    close(torch.cat(got), wanted(name, t), dtype)


@pytest.mark.parametrize("name", list(CONFIGS_8))
def test_many_rows(name):
    """A step whose rows take the kernels for many rows gives what portions give."""
    cfg, m = model(name, BF16)
    t = prompt(700, cfg["vocab"], 3)
    a = engine(m, graphs=False).feed([("a", t, list(range(600, 700)))])
    e, b = engine(m, graphs=False), None
    for i in range(0, 700, 100):
        b = e.feed([("a", t[i:i + 100], list(range(100)))])
    close(a, b.cpu(), BF16)


@pytest.mark.parametrize("name", ["wide", "both"])
def test_captured_decoding_and_mixed_steps(name):
    """Decoding steps are replayed from graphs; the same tokens without them, in another batch, give the same ones."""
    from atma_b200.engine import SamplingParams
    cfg, m = model(name, F32)
    prompts = [prompt(n, cfg["vocab"], 30 + n) for n in (3, 20, 1, 33)]
    a = engine(m, max_step_tokens=24, block_size=16).generate(prompts, SamplingParams(max_new_tokens=8))
    b = [engine(m, graphs=False, block_size=16).generate([p], SamplingParams(max_new_tokens=8))[0] for p in prompts]
    for x, y, p in zip(a, b, prompts):
        logits = wanted(name, p + y[:-1])[len(p) - 1:]
        top = logits.topk(2, -1).values
        clear = ((top[:, 0] - top[:, 1]) > 0.2 * logits.std()).tolist()                        # beyond what values over borders change
        upto = next((i for i, (c, u, v) in enumerate(zip(clear, x, y)) if u != v), len(x))
        assert upto == len(x) or not clear[upto]
        assert all(int(l.argmax()) == v for l, v, c in zip(logits, y, clear) if c)


def test_a_folder_with_experts(tmp_path, capsys):
    """The command that generates takes such a folder; weights in 8 bits are named by config.json."""
    from atma_b200 import checkpoint, generate
    from atma_b200.engine import SamplingParams
    cfg, m = model("both", BF16)
    checkpoint.write_model(tmp_path / "m", cfg, {n: t.bfloat16() for n, t in O.rizurax_weights(cfg, 7).items()})
    assert json.loads((tmp_path / "m" / "config.json").read_text())["weights"] == "e4m3"
    p = prompt(11, cfg["vocab"], 5)
    want = engine(m).generate([p], SamplingParams(max_new_tokens=5))[0]
    generate.main(["--model", str(tmp_path / "m"), "--prompt", ",".join(map(str, p)), "--max-new-tokens", "5", "--max-tokens", "600"])
    assert capsys.readouterr().out.strip() == ",".join(map(str, want))
