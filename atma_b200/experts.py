"""Mixtures of experts (libatma_decoder.so): which experts a token goes to, and their feed-forwards in 8 bits.

    routes = route_experts(logits, top_k, score="sigmoid", bias=balance, groups=8, top_groups=4)
    y = expert_mlp(rows, w_gate_up, w_down, routes)

All launches have shapes that the host knows (tokens x top_k rows), so that a step with experts can be captured in a CUDA graph.
"""

import ctypes

import torch

from . import _lib
from .decoder_ops import _check
from .fp8_ops import Fp8Rows, Fp8Weight, _here, _new, _stream, _TYPES

MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 512, 64, 64
_EXACT = (torch.float32, torch.bfloat16, torch.float16)       # what float32, which a choice is made from, holds without rounding


class Routes:
    """Where tokens go.  ids, weights (tokens, top_k): experts (int32) and their weights (float32), the best first.  A pair
    token * top_k + choice is a row of the experts' products: order[row] = pair (rows by expert, then by pair), place[pair] = row,
    and expert e's rows are starts[e] .. starts[e + 1] - 1 (all int32).  weights may be replaced by others of the same shape; ids are what the
    places were made from."""

    __slots__ = ("ids", "weights", "experts", "_plan")

    def __init__(self, ids, weights, experts, plan):
        self.ids, self.weights, self.experts, self._plan = ids, weights, experts, plan          # plan: order, place and starts, one behind another

    @property
    def order(self):
        return self._plan[:self.ids.numel()]

    @property
    def place(self):
        n = self.ids.numel()
        return self._plan[n:2 * n]

    @property
    def starts(self):
        return self._plan[2 * self.ids.numel():]


def route_experts(logits, top_k, *, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """Experts of tokens by their logits (tokens, experts), float32 or 16-bit.  ``score``: "softmax" or "sigmoid"; a choice goes by score +
    ``bias`` (experts,), float32 or 16-bit, weights by the scores alone.  ``groups``: of so many groups of neighbouring experts only ``top_groups`` are
    looked at, those with the largest sum of their two best (None: all).  ``renormalize``: a token's weights are divided by their sum (zero where that is
    zero); ``scale`` multiplies them.  Equal ones: the lower index first.  NaN and -inf count as the least finite logit, inf as the
    largest; a choice is decided as in 64-bit arithmetic, and scores too small for fp32 are divided in it."""
    here, shape = _here(logits, bias), logits.shape
    if len(shape) != 2 or logits.dtype not in _EXACT:
        raise ValueError("logits must be a (tokens, experts) matrix of float32, bfloat16 or float16")
    (tokens, experts), dev = shape, logits.device
    if top_groups is None:
        top_groups = groups
    if score != "softmax" and score != "sigmoid":
        raise ValueError(f"unknown score {score!r}; expected 'softmax' or 'sigmoid'")
    if not 0 < experts <= MAX_EXPERTS or not 0 < groups <= MAX_GROUPS or experts % groups or not 0 < top_groups <= groups:
        raise ValueError(f"{top_groups} of {groups} groups of {experts} experts (at most {MAX_EXPERTS} in {MAX_GROUPS} groups)")
    if not 0 < top_k <= min(MAX_TOP_K, experts // groups * top_groups):
        raise ValueError(f"{top_k} of {experts // groups * top_groups} experts (at most {MAX_TOP_K})")
    step, unit = logits.stride()
    if logits.dtype is not torch.float32 or unit != 1 and experts > 1 or step < experts and tokens > 1:
        logits, step = logits.float().contiguous(), experts
    if bias is not None:
        if bias.shape != (experts,) or bias.dtype not in _EXACT:
            raise ValueError(f"bias must have {experts} values of float32, bfloat16 or float16, not the shape {tuple(bias.shape)} of {bias.dtype}")
        if bias.dtype is not torch.float32 or not bias.is_contiguous():
            bias = bias.float().contiguous()
    lib, n, i32 = _lib.load_decoder(), tokens * top_k, torch.int32
    ids = _new((tokens, top_k), (top_k, 1), device=dev, dtype=i32)
    weights = _new((tokens, top_k), (top_k, 1), device=dev, dtype=torch.float32)
    plan = _new((2 * n + experts + 1,), (1,), device=dev, dtype=i32)
    ints, at = lib.atma_route_scratch_ints(tokens, experts), plan.data_ptr()
    scratch = _new((ints,), (1,), device=dev, dtype=i32) if ints else None
    rc = lib.atma_route_experts(logits.data_ptr(), step if tokens > 1 else experts, None if bias is None else bias.data_ptr(), ids.data_ptr(),
                                weights.data_ptr(), at, at + 4 * n, at + 8 * n, None if scratch is None else scratch.data_ptr(), tokens, experts, top_k,
                                score == "sigmoid", groups, top_groups, bool(renormalize), scale, _stream(here))
    if rc:
        _check(rc)
    return Routes(ids, weights, experts, plan)


def expert_mlp(x, w_gate_up, w_down, routes, add=None, dtype=torch.bfloat16):
    """Gelu-gated feed-forwards of the tokens' experts, weighted and summed: sum over j of weights[t, j] * down(gelu_tanh(gate x_t) * up x_t).
    x: Fp8Rows (tokens, width); w_gate_up (experts, 2, ff, width), w_down (experts, width, ff): Fp8Weight; the activations between them go
    to 8 bits like any rows.  ``add`` (tokens, width) is added.  Returns (tokens, width) in ``dtype``, bfloat16 or float32; the sum
    is fp32, and so is what is summed."""
    if not isinstance(x, Fp8Rows) or not isinstance(w_gate_up, Fp8Weight) or not isinstance(w_down, Fp8Weight) or not isinstance(routes, Routes):
        raise ValueError("expert_mlp takes Fp8Rows, two Fp8Weights and Routes")
    (tokens, width), (chosen, top_k), experts = x.values.shape, routes.ids.shape, routes.experts
    ff = w_down.values.shape[-1]
    if w_gate_up.values.shape != (experts, 2, ff, width) or w_down.values.shape != (experts, width, ff) or chosen != tokens:
        raise ValueError(f"weights of the shapes {tuple(w_gate_up.shape)} and {tuple(w_down.shape)} do not fit rows {tuple(x.shape)} and "
                         f"{tuple(routes.ids.shape)} choices of {experts} experts")
    if routes.weights.shape != routes.ids.shape or routes.weights.dtype is not torch.float32 or not routes.weights.is_contiguous():
        raise ValueError("the routes' weights must be (tokens, top_k) float32, contiguous")
    plan = routes._plan                          # other ids than route_experts gave have other places: rows would be written behind the scratch memory
    if plan.shape != (2 * tokens * top_k + experts + 1,) or plan.dtype is not torch.int32 or not plan.is_contiguous():
        raise ValueError(f"the routes' places are not those of {tokens} tokens with {top_k} of {experts} experts: another choice takes another call of route_experts")
    if dtype not in _TYPES or add is not None and (add.shape != (tokens, width) or add.dtype is not dtype or not add.is_contiguous()):
        raise ValueError("bfloat16 or float32, add contiguous in the same type")
    here, dev = _here(x.values, w_gate_up.values, w_down.values, plan, routes.weights, add), x.values.device
    lib, code = _lib.load_decoder(), _lib.DTYPE_CODE[dtype]
    out = _new((tokens, width), (width, 1), device=dev, dtype=dtype)
    scratch = _new((lib.atma_expert_mlp_scratch_bytes(tokens, top_k, width, ff, code),), (1,), device=dev, dtype=torch.uint8)
    place = plan.data_ptr() + 4 * tokens * top_k
    a = _lib.ExpertArgs(x.values.data_ptr(), x.row_stride, x.scales.data_ptr(), x.scale_stride, w_gate_up.values.data_ptr(), w_gate_up.row_stride,
                        w_gate_up.scales.data_ptr(), w_down.values.data_ptr(), w_down.row_stride, w_down.scales.data_ptr(), place, place + 4 * tokens * top_k,
                        routes.weights.data_ptr(), None if add is None else add.data_ptr(), out.data_ptr(), tokens, top_k, experts, width, ff, code)
    rc = lib.atma_expert_mlp(ctypes.byref(a), scratch.data_ptr(), _stream(here))
    if rc:
        _check(rc)
    return out
