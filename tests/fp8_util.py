"""Small configurations with projections in 8 bits and with experts, for the host and the GPU tests."""

from tests.rizurax_util import attention, config, delta


def experts(layer, n, top_k, ff, **kw):
    return {**layer, "mlp": {"kind": "experts", "experts": n, "top_k": top_k, "ff": ff, **kw}}


CONFIGS_8 = {
    # every kind of layer in 8 bits; no width is a multiple of a block
    "dense": {**config([attention(6, 2, 12, 20, rot=8, ff=56), delta(6, 3, 20, 12, conv=3), attention(2, 1, 24, 8, rot=24, ff=None), delta(2, 2, 8, 36, conv=2, ff=300)],
                       loop=(1, 3, 2)), "weights": "e4m3"},
    # head sizes of the tensor-core kernels, several blocks
    "wide": {**config([delta(4, 2, 128, 128, conv=4, ff=256), attention(4, 2, 64, 128, rot=32, base=5000.0, ff=192)], vocab=160, width=384), "weights": "e4m3"},
    # experts between other layers, projections in the model's own type
    "experts": config([experts(attention(4, 2, 16, 20), 6, 2, 72), delta(2, 1, 16, 24, ff=40), experts(delta(3, 3, 12, 16), 9, 3, 130, score="sigmoid", renormalize=False, scale=1.5)],
                      width=96),
    # both, with a bias, groups, and a looped layer of experts
    "both": {**config([experts(attention(4, 2, 16, 32), 16, 3, 128, score="sigmoid", bias=True, groups=4, top_groups=2), delta(2, 1, 16, 24, ff=136)], width=128, loop=(0, 1, 2),
                      bigram=None), "weights": "e4m3"},
}
