"""Rizurax: a decoder-only language model whose layers each hold a token mixer (gated delta rule or differential
attention) and, optionally, a gelu-gated feed-forward, both fed by their own norm of the same residual stream:

    x <- x + mixer(norm1(x)) + ff(norm2(x))

A stretch of layers may run several times in a row with the same weights; every pass has its own cache or state.  The
embedding adds a hashed bigram term.  The residual stream is fp32.

config.json: ``vocab``, ``width``, ``norm.eps``, ``embedding.bigram`` (buckets, mul_prev, mul_cur), ``layers`` (type,
mixer sizes, mlp or null) and ``loop`` (start, stop, times).  Tensors: embed, bigram, l<i>.norm1/2, l<i>.mix.*,
l<i>.mlp.gate/up/down, final.norm, head.

A layer's mixer output and its feed-forward activation lie side by side in one buffer, so that W_o and W_down are one
matrix product whose sum is what the residual stream receives; the add, the next layer's two norms and the conversion
of their results are one launch.

``"weights": "e4m3"`` in config.json: the layers' projections are products in 8 bits (``fp8_ops``; weights are converted when the
model is loaded, norms hand out rows in 8 bits, and so does the feed-forward's first product).  A feed-forward of ``"kind":
"experts"`` (ff, experts, top_k; optional score, bias, groups, top_groups, renormalize, scale: ``experts.route_experts``) has tensors
l<i>.mlp.router (experts, width), l<i>.mlp.router.bias (experts,) with ``"bias": true``, and gate, up (experts, ff, width) and down
(experts, width, ff); its experts' weights are in 8 bits in either case.
"""

from types import SimpleNamespace

import torch

from . import decoder_ops as ops
from . import fp8_ops as ops8
from .configured import ConfiguredModel
from .experts import expert_mlp, route_experts
from .mixers import GatedDelta, SoftmaxAttention

UNIT_EPS = 1e-6                # inside the root of the unit vectors of q and k


def layer_order(config):
    """Layer index of every layer run, looped stretches unrolled."""
    n, loop = len(config["layers"]), config.get("loop")
    if not loop:
        return list(range(n))
    start, stop, times = loop["start"], loop["stop"], loop["times"]
    if not 0 <= start <= stop <= n or times < 0:
        raise ValueError(f"loop {loop} does not fit {n} layers")
    return list(range(start)) + list(range(start, stop)) * times + list(range(stop, n))


class RizuraxModel(ConfiguredModel):
    def _build(self, config):
        self.order = layer_order(config)
        if config.get("weights") not in (None, "e4m3"):
            raise ValueError(f"unknown weights {config['weights']!r}; this model has them in its own type or in \"e4m3\"")
        self.in_8_bits = config.get("weights") == "e4m3"
        self.embed = self._w("embed", self.vocab, self.width)
        big = (config.get("embedding") or {}).get("bigram")
        self.bigram = self._w("bigram", big["buckets"] + 1, self.width) if big else None
        self.bigram_mul = (big["mul_prev"], big["mul_cur"]) if big else (0, 0)
        self.layers = [self._layer(i, e) for i, e in enumerate(config["layers"])]
        self.final_norm, self.head = self._w("final.norm", self.width), self._w("head", self.vocab, self.width)
        self.run_mixers = [self.layers[i].mixer for i in self.order]           # a looped layer has a cache per pass

    # ---- weights ----------------------------------------------------------------------------------------------
    def _layer(self, i, entry):
        p, D, m = f"l{i}.", self.width, entry["mixer"]
        kind = entry["type"]
        if kind == "attention":
            mixer = self._attention(p + "mix.", m)
        elif kind == "delta":
            mixer = self._delta(p + "mix.", m)
        else:
            raise ValueError(f"layer {i}: unknown mixer {kind!r}")
        layer = SimpleNamespace(mixer=mixer, norm1=self._w(p + "norm1", D), norm2=None, w_gate_up=None, ff=0, experts=None)
        w_out, mlp = [self._w(p + "mix.o", D, mixer.width)], entry.get("mlp")
        layer.mixed = mixer.width                    # where the feed-forward's activations begin beside the mixer's results
        if self.in_8_bits:
            mixer.w_in = ops8.Fp8Weight.of(mixer.w_in)
            layer.mixed += -mixer.width % ops8.BLOCK
        if mlp is not None:
            layer.norm2 = self._w(p + "norm2", D)
            if mlp.get("kind", "dense") == "experts":
                layer.experts = self._experts(p + "mlp.", mlp)
            elif mlp.get("kind", "dense") == "dense":
                layer.ff = mlp["ff"]
                gate_up = [self._w(p + "mlp.gate", layer.ff, D), self._w(p + "mlp.up", layer.ff, D)]
                layer.w_gate_up = ops8.Fp8Weight.of(torch.stack(gate_up)) if self.in_8_bits else torch.cat(gate_up).contiguous()
                w_out += [w_out[0].new_zeros(D, layer.mixed - mixer.width), self._w(p + "mlp.down", D, layer.ff)]
            else:
                raise ValueError(f"layer {i}: unknown feed-forward {mlp['kind']!r}")
        layer.w_out = torch.cat(w_out, dim=1).contiguous()
        if self.in_8_bits:
            layer.w_out = ops8.Fp8Weight.of(layer.w_out)
        return layer

    def _experts(self, p, m):
        D, n, ff = self.width, m["experts"], m["ff"]
        of = ops8.Fp8Weight.of
        return SimpleNamespace(router=self._w(p + "router", n, D), top_k=m["top_k"], ff=ff,
                               w_gate_up=of(torch.stack([self._w(p + "gate", n, ff, D), self._w(p + "up", n, ff, D)], 1)), w_down=of(self._w(p + "down", n, D, ff)),
                               options=dict(score=m.get("score", "softmax"), groups=m.get("groups", 1), top_groups=m.get("top_groups"),
                                            renormalize=m.get("renormalize", True), scale=float(m.get("scale", 1.0)),
                                            bias=self._w(p + "router.bias", n, dtype=torch.float32) if m.get("bias") else None))

    def _attention(self, p, m):
        D, H, G, d, e = self.width, m["heads"], m["kv_heads"], m["dim"], m["vdim"]
        diff = float(m["diff"])
        lq1, lk1, lq2, lk2 = (self._w(p + n, d, dtype=torch.float32) for n in ("lq1", "lk1", "lq2", "lk2"))
        lam = float(torch.exp((lq1 * lk1).sum()) - torch.exp((lq2 * lk2).sum()) + diff)
        return SoftmaxAttention(self._w(p + "q", H * 2 * d, D), self._w(p + "k", G * 2 * d, D), self._w(p + "v", G * e, D), heads=H,
                                kv_heads=G, maps=2, dim=d, vdim=e, scale=float(m["scale"]), rotary=self._rotary(m.get("rot")), lam=lam,
                                out_scale=1.0 - diff, eps=self.eps)

    def _delta(self, p, m):
        D, H, G, d, e, taps = self.width, m["heads"], m["kv_heads"], m["dim"], m["vdim"], m["conv"]
        f32 = torch.float32
        weights = ops.DeltaWeights(self._w(p + "q.conv", G * d, taps), self._w(p + "k.conv", G * d, taps), self._w(p + "v.conv", H * e, taps),
                                   self._w(p + "A_log", H, dtype=f32), self._w(p + "dt_bias", H, dtype=f32), self._w(p + "norm", e), heads=H,
                                   kv_heads=G, dim=d, vdim=e, unit_eps=UNIT_EPS, q_scale=d ** -0.5)
        return GatedDelta(self._w(p + "q", G * d, D), self._w(p + "k", G * d, D), self._w(p + "v", H * e, D), self._w(p + "g", H * e, D),
                          self._w(p + "a", H, D), self._w(p + "b", H, D), weights, self.eps)

    # ---- the step ---------------------------------------------------------------------------------------------
    def _norms(self, x, y, layer):
        """What a layer reads, after x += y: its mixer's rows and its feed-forward's (None without one); for experts the latter as
        (rows in 8 bits, the same in the activation dtype)."""
        weights, routed = (layer.norm1, layer.norm2), layer.experts is not None
        if self.in_8_bits:
            (h1, _), (h2, plain) = ops8.residual_norms_fp8(x, y, weights, self.eps, plain=routed)
        else:
            h1, plain = ops.residual_norms(x, y, weights, self.eps)
            h2 = ops8.quantize_rows(plain) if routed else plain
        return h1, (h2, plain) if routed else h2

    def _layer_run(self, layer, h1, h2, batch, state):
        """What the layer adds to the residual stream."""
        n, width, dev = batch.ids.shape[0], layer.mixer.width, self.device
        if not self.in_8_bits:
            act = torch.empty((n, width + layer.ff), device=dev, dtype=self.dtype)
            layer.mixer.run(h1, act[:, :width], batch, state)
            if layer.ff:
                ops.gelu_gated_linear(h2, layer.w_gate_up, act[:, width:])
        else:
            mixed = torch.empty((n, width), device=dev, dtype=self.dtype)
            layer.mixer.run(h1, mixed, batch, state)
            if layer.ff:
                act = ops8.empty_rows(n, layer.mixed + layer.ff, dev)
                if layer.mixed > width:
                    act.values[:, width:layer.mixed].zero_()                       # they meet zeros of the weight
                ops8.quantize_rows(mixed, out=act.columns(0, layer.mixed, width))
                ops8.gelu_gated_linear_fp8(h2, layer.w_gate_up, out=act.columns(layer.mixed, layer.mixed + layer.ff))
            else:
                act = ops8.quantize_rows(mixed)
        y = ops.linear(act, layer.w_out, dtype=self.dtype)
        if layer.experts is not None:
            e, (rows, plain) = layer.experts, h2
            routes = route_experts(ops.linear_f32_out(plain, e.router), e.top_k, **e.options)
            y = expert_mlp(rows, e.w_gate_up, e.w_down, routes, add=y, dtype=self.dtype)
        return y

    @torch.no_grad()
    def forward(self, batch, state, record=None):
        """One step: the batch's rows through all layers, caches and states updated; fp32 logits of ``batch.logit_rows``
        (None when empty).  ``record``: a list that receives the residual stream after every layer run."""
        x = ops.embed_bigram(batch.ids, batch.prev, self.embed, self.bigram, *self.bigram_mul)
        runs = [self.layers[i] for i in self.order]
        h1, h2 = self._norms(x, None, runs[0]) if runs else (None, None)
        y = None
        for r, layer in enumerate(runs):
            y = self._layer_run(layer, h1, h2, batch, state[r])
            if r + 1 < len(runs):
                h1, h2 = self._norms(x, y, runs[r + 1])
                if record is not None:
                    record.append(x.clone())
        if record is not None and y is not None:
            record.append(x + y)
        if batch.logit_rows is None:
            return None
        xs, ys = x.index_select(0, batch.logit_rows), None if y is None else y.index_select(0, batch.logit_rows)
        h, = ops.residual_norms(xs, ys, (self.final_norm,), self.eps)
        return ops.linear_f32_out(h, self.head)

    def weight_bytes(self):
        """Bytes of weights one decode step reads (a looped layer's once per pass; of experts all, which many sequences reach)."""
        size = lambda w: 0 if w is None else w.nbytes() if isinstance(w, ops8.Fp8Weight) else w.numel() * w.element_size()
        parts = lambda l: [l.mixer.w_in, l.w_out, l.w_gate_up] + ([] if l.experts is None else [l.experts.router, l.experts.w_gate_up, l.experts.w_down])
        return sum(size(w) for i in self.order for w in parts(self.layers[i])) + size(self.head)
