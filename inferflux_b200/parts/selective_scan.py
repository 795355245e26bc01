"""A mixer whose state decays at a rate of its own for every channel and every number of the state, chosen by the input:

    [x | z] = W_in h;   x <- silu(conv(x) + b_conv)                          (causal, per channel, over time)
    [s | B | C] = W_x x                                                     (each over its root mean square times a weight, with `norms`)
    step = softplus(W_dt s + b_dt),   A = -exp(A_log)                        [channels, states]
    h[c, n] <- exp(step[c] A[c, n]) h[c, n] + step[c] x[c] B[n]
    y = W_o ((sum_n C[n] h[c, n] + D[c] x[c]) * silu(z))

The convolution's last taps - 1 input rows and h (float32) are the request's state.  W_in's, the convolution's and W_o's rows are in the
run's dtype; W_x and W_dt hand their results over in float32, and steps, decays, h and the sums over it are float32.
"""
from __future__ import annotations

import torch

from ..weights.loader import TensorSpec
from .attention import materialized_rows
from .base import Mixer, StateSpec, WeightBuffers, register_part


@register_part("mixer", "selective_state_space")
class SelectiveStateSpace(Mixer):
    """params: hidden_size, inner_size, state_dim, step_rank, conv_taps, norms (whether s, B and C are normed; default False), norm_eps,
    names (tensor names of in, conv, conv_bias, x, dt, dt_bias, A_log, D, o and, with norms, dt_norm, b_norm, c_norm)."""

    _NAMES = {"in": "in", "conv": "conv", "conv_bias": "conv.b", "x": "x", "dt": "dt", "dt_bias": "dt.b", "A_log": "A_log", "D": "D", "o": "o",
              "dt_norm": "dt_norm", "b_norm": "b_norm", "c_norm": "c_norm"}

    def __init__(self, spec):
        super().__init__(spec)
        p = spec.params
        self.hidden, self.inner = int(p["hidden_size"]), int(p["inner_size"])
        self.n, self.rank, self.taps = int(p["state_dim"]), int(p["step_rank"]), int(p["conv_taps"])
        if min(self.hidden, self.inner, self.n, self.rank, self.taps) <= 0:
            raise ValueError("selective_state_space: sizes must be positive")
        if self.n > 128 or self.taps > 16 or self.rank > 8192:
            raise ValueError("selective_state_space: a state of more than 128, more than 16 taps or a rank above 8,192 is beyond the kernels")
        self.norms = bool(p.get("norms", False))
        self.eps = float(p.get("norm_eps", 1e-6))
        self.names = dict(self._NAMES)
        self.names.update(p.get("names") or {})
        self.norm_weights = None

    def state_spec(self):
        """[the convolution's last taps - 1 input rows, then h as [channel, state number]]."""
        return StateSpec(((self.taps - 1 + self.n) * self.inner,), torch.float32)

    def _vectors(self):
        out = {"conv_bias": (self.inner, "zeros"), "dt_bias": (self.inner, "zeros"), "D": (self.inner, "ones")}
        if self.norms:
            out.update({"dt_norm": (self.rank, "ones"), "b_norm": (self.n, "ones"), "c_norm": (self.n, "ones")})
        return out

    def param_specs(self):
        n, C, H = self.names, self.inner, self.hidden
        specs = {n["in"]: TensorSpec((2 * C, H)), n["conv"]: TensorSpec((C, self.taps)), n["x"]: TensorSpec((self.rank + 2 * self.n, C)),
                 n["dt"]: TensorSpec((C, self.rank)), n["A_log"]: TensorSpec((C, self.n), init="zeros"), n["o"]: TensorSpec((H, C))}
        specs.update({n[s]: TensorSpec((size,), init=init) for s, (size, init) in self._vectors().items()})
        return specs

    def load(self, tensors, dtype, device):
        n, C, H, f32 = self.names, self.inner, self.hidden, torch.float32
        layout = {"in": ((2 * C, H), dtype), "x": ((self.rank + 2 * self.n, C), dtype), "dt": ((C, self.rank), dtype), "o": ((H, C), dtype),
                  "conv": ((C, self.taps), f32), "A_log": ((C, self.n), f32)}
        layout.update({s: ((size,), f32) for s, (size, _init) in self._vectors().items()})
        self.buffers = buf = WeightBuffers(device, layout)
        for s in layout:
            buf[s].copy_(tensors[n[s]])
        self.norm_weights = (buf["dt_norm"], buf["b_norm"], buf["c_norm"]) if self.norms else None

    def forward(self, h, ctx, cache):
        k, buf, C, f32 = ctx.kernels, self.buffers, self.inner, torch.float32
        rows = (self.taps - 1) * C
        xz = k.linear(materialized_rows(k, h), buf["in"])                                                  # [T, x | z]
        conv_state = None if self.taps < 2 else cache.state[:, :rows].unflatten(1, (1, self.taps - 1, C))
        x = k.short_conv(xz, buf["conv"], self.taps, conv_state, 0, ctx, add_input=False, bias=buf["conv_bias"], act="silu", columns=(0, C))
        low, bc = k.selective_inputs(k.linear(x, buf["x"], out_dtype=f32, allow_partial=True), self.rank, self.n, ctx.dtype,
                                     norms=self.norm_weights, eps=self.eps)
        y = k.selective_scan(x, k.linear(low, buf["dt"], out_dtype=f32), bc, buf["A_log"], cache.state[:, rows:], ctx, z=xz[:, C:],
                             bias=buf["dt_bias"], skip=buf["D"], out_dtype=ctx.dtype)
        return k.linear(y, buf["o"], allow_partial=True)
