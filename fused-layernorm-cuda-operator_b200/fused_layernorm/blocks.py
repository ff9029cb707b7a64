"""The norms around a transformer block and inside its attention, fused with what stands next to
them.  The reference has none of these; they are siblings of the residual-add norms in
rmsnorm.py.

  fused_norm_gate_add_norm   the norm behind a block, the block's gate and scale, the residual
                             add, and the norm in front of the next block
  fused_qk_norm_rotary       the norm of every q and k head and the rotation of rotary positions
                             with one or several axes (time, height, width)

Both take fp32, bf16 and fp16 CUDA tensors, keep everything between their inputs and outputs in
32 bits, are differentiable (one C++ autograd node each; second and forward-mode derivatives are
refused), launch on the current stream, can be captured into a CUDA graph, and trace under
torch.compile, apart from fused_qk_norm_rotary_, which breaks the graph there and runs between its
parts.  As with every autograd function, capturing a backward pass needs leaves whose gradients no
eager graph still refers to.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
from torch.nn import Parameter

import fused_layernorm_cuda as _ext

from . import ops as _ops
from .layernorm import _require_cuda

_t = torch.ops.fused_layernorm
_KINDS = {"layernorm": _ops.LAYERNORM, "rmsnorm": _ops.RMSNORM, "none": _ops.NO_NORM}
_ACTS = {"none": 0, "sigmoid": 1, "silu": 2, "tanh": 3}
_LAYOUTS = {"half": 0, "interleaved": 1}


def _choice(table, value, name):
    try:
        return table["none" if value is None else value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {', '.join(map(repr, table))}, got {value!r}") from None


def fused_norm_gate_add_norm(input: torch.Tensor, residual: Optional[torch.Tensor] = None,
                             gate: Optional[torch.Tensor] = None, post_weight: Optional[torch.Tensor] = None,
                             post_bias: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                             bias: Optional[torch.Tensor] = None, *, post_norm: Optional[str] = "rmsnorm",
                             norm: Optional[str] = "rmsnorm", gate_activation: Optional[str] = "none",
                             branch_scale: float = 1.0, residual_scale: float = 1.0, weight_offset: float = 0.0,
                             post_eps: float = 1e-6, eps: float = 1e-6) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """(y, sum) of
        sum = residual_scale * residual + branch_scale * act(gate) * N1(input)
        y   = N2(sum)
    in one pass over HBM, over the last dimension of an input of any rank.  N1 (`post_norm`, the
    norm behind the block) and N2 (`norm`, the one in front of the next block) are "rmsnorm",
    "layernorm" or "none", scaled by (weight_offset + weight) and shifted by bias where those are
    given.  `norm="none"` returns (None, sum).  residual and gate may be absent; act is "none",
    "sigmoid", "silu" or "tanh" (without a gate there is nothing for it to act on).

    gate is [hidden], one vector for each entry of the first dimension
    ([input.shape[0], hidden], also with dimensions of size one in between), or of the shape of
    input; weight and bias are [hidden] or one vector for each entry of the first dimension (with
    weight_offset=1 that is adaptive modulation, (1 + scale) and shift per sample; the offset is
    that of both norms).

    The sum stays in 32 bits for N2 and is rounded only where it is returned, so y may differ in
    its last bit from a norm taken of the returned sum.  Differentiable in all seven tensors; the
    gradient that arrives on the returned sum is taken in by the same backward kernel.  All
    tensors share one dtype."""
    post_kind, kind = _choice(_KINDS, post_norm, "post_norm"), _choice(_KINDS, norm, "norm")
    act = _choice(_ACTS, gate_activation, "gate_activation")
    _require_cuda(input)
    conf = (post_kind, kind, act, float(branch_scale), float(residual_scale), float(weight_offset), float(post_eps),
            float(eps))
    if not torch.compiler.is_compiling():
        return _ext.norm_gate_add_norm(input, residual, gate, post_weight, post_bias, weight, bias, *conf)
    y, s, *_stats = _t.norm_gate_add_norm_fwd(input, residual, gate, post_weight, post_bias, weight, bias, *conf)
    return (y if kind != _ops.NO_NORM else None), s


class FusedNormGateAddNorm(nn.Module):
    """fused_norm_gate_add_norm with its parameters: `post_weight` / `post_bias` of the norm behind
    the block, `weight` / `bias` of the norm in front of the next one (biases with bias=True, for
    layer norms), and with layer_scale a learned `gate` of [hidden] that starts at that value.
    Weights start at one, or at zero with weight_offset=1 (weights stored around zero).

        y, residual = m(block_output, residual)          # m(block_output, residual, gate=g): another gate
    """

    def __init__(self, hidden: int, post_norm: Optional[str] = "rmsnorm", norm: Optional[str] = "rmsnorm",
                 bias: bool = False, layer_scale: Optional[float] = None, gate_activation: Optional[str] = "none",
                 branch_scale: float = 1.0, residual_scale: float = 1.0, weight_offset: float = 0.0,
                 post_eps: float = 1e-6, eps: float = 1e-6, elementwise_affine: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        self.hidden, self.post_norm, self.norm = int(hidden), post_norm or "none", norm or "none"
        _choice(_KINDS, self.post_norm, "post_norm"), _choice(_KINDS, self.norm, "norm")
        _choice(_ACTS, gate_activation, "gate_activation")
        self.gate_activation = gate_activation or "none"
        self.branch_scale, self.residual_scale, self.weight_offset = branch_scale, residual_scale, weight_offset
        self.post_eps, self.eps = post_eps, eps

        def parameter(present, value):
            return Parameter(torch.full((self.hidden,), float(value), device=device, dtype=dtype)) if present else None

        has1, has2 = self.post_norm != "none" and elementwise_affine, self.norm != "none" and elementwise_affine
        self.register_parameter("post_weight", parameter(has1, 1.0 - weight_offset))
        self.register_parameter("post_bias", parameter(has1 and bias, 0.0))
        self.register_parameter("weight", parameter(has2, 1.0 - weight_offset))
        self.register_parameter("bias", parameter(has2 and bias, 0.0))
        self.register_parameter("gate", parameter(layer_scale is not None, layer_scale or 0.0))

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None):
        gate = self.gate if gate is None else gate
        return fused_norm_gate_add_norm(input, residual, gate, self.post_weight, self.post_bias, self.weight, self.bias,
                                        post_norm=self.post_norm, norm=self.norm,
                                        gate_activation=self.gate_activation,
                                        branch_scale=self.branch_scale, residual_scale=self.residual_scale,
                                        weight_offset=self.weight_offset, post_eps=self.post_eps, eps=self.eps)

    def extra_repr(self) -> str:
        return "{hidden}, post_norm={post_norm!r}, norm={norm!r}, gate_activation={gate_activation!r}".format(**self.__dict__)


# ------------------------------------------------------------------------------------ rotary
# 2**192 / (2 pi)
_TURN = 0x28be60db9391054a7f09d5f47d4d377036d8a5664f10e410


def _turns(inv_freq: float) -> int:
    """inv_freq / (2 pi) as a 64-bit binary fraction of a turn, as a signed 64-bit integer."""
    num, den = inv_freq.as_integer_ratio()  # den is a power of two
    n = ((num * _TURN) >> (126 + den.bit_length())) + 1 >> 1  # rounded to nearest
    n %= 1 << 64
    return n - (1 << 64) if n >= 1 << 63 else n


class RotaryAxes:
    """The rotary plan of a model: which pair of a head's elements turns with which axis, and how
    fast.  A program makes it once.

        RotaryAxes(128, 64)                              # one axis, all 64 pairs
        RotaryAxes(128, (16, 24, 24), base=1e6)          # time, height, width along one ladder
        RotaryAxes(72, (12, 12, 12), per_axis=True)      # a ladder of its own for each axis
        RotaryAxes(128, 32)                              # rotates the first 64 elements only

    sections: pairs for each axis; 2 * sum(sections) <= head_dim elements are rotated, the ones
    behind them are left as the norm made them.  Pair i (counted over all sections, or within its
    section with per_axis) has inv_freq = base ** (-i / n) with n = sum(sections), or the
    section's size with per_axis; inv_freq gives the frequencies of all pairs instead (float64
    values).  interleaved_axes deals the pairs out in turn (pair 0 to axis 0, pair 1 to axis 1,
    ...) until an axis has its share, instead of section by section.  position_scale, one number
    per axis, multiplies the positions.  layout: "half" pairs element i with i + sum(sections),
    "interleaved" pairs 2i with 2i + 1.  magnitude multiplies the rotated elements.

    Positions are whole numbers; the angle position * inv_freq is reduced exactly (to
    |position| * 2**-65 turns) and rounded to 32 bits only behind its whole quarter turns, so far
    positions lose nothing and a cosine or sine is good to some 2**-22 of itself."""

    def __init__(self, head_dim: int, sections: Union[int, Sequence[int]], base: float = 10000.0, *,
                 per_axis: bool = False, layout: str = "half", inv_freq: Optional[Sequence[float]] = None,
                 interleaved_axes: bool = False, position_scale: Optional[Sequence[float]] = None,
                 magnitude: float = 1.0, device="cuda") -> None:
        sections = (int(sections),) if isinstance(sections, int) else tuple(int(n) for n in sections)
        pairs = sum(sections)
        if not sections or min(sections) < 0 or len(sections) > 255:
            raise ValueError(f"sections must be pair counts, one for each axis, got {sections}")
        if 2 * pairs > head_dim:
            raise ValueError(f"sections {sections} rotate {2 * pairs} elements, more than head_dim {head_dim}")
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if position_scale is not None and len(position_scale) != len(sections):
            raise ValueError("position_scale needs one number for each axis")
        if inv_freq is None and not (base > 0 and math.isfinite(base)):
            raise ValueError(f"base must be positive, got {base}")
        self.head_dim, self.sections, self.layout, self.magnitude = int(head_dim), sections, layout, float(magnitude)
        self.axes, self.pairs = len(sections), pairs
        if interleaved_axes:
            left, axis = list(sections), []
            while len(axis) < pairs:
                for a in range(len(sections)):
                    if left[a] > 0:
                        axis.append(a)
                        left[a] -= 1
        else:
            axis = [a for a, n in enumerate(sections) for _ in range(n)]
        if inv_freq is None:
            seen, freq = [0] * len(sections), []
            for i, a in enumerate(axis):
                freq.append(float(base) ** (-(seen[a] / sections[a] if per_axis else i / pairs)))
                seen[a] += 1
        else:
            freq = [float(f) for f in inv_freq]
            if len(freq) != pairs:
                raise ValueError(f"inv_freq needs {pairs} values, got {len(freq)}")
        if position_scale is not None:
            freq = [f * float(position_scale[a]) for f, a in zip(freq, axis)]
        if not all(math.isfinite(f) for f in freq):
            raise ValueError("frequencies must be finite")
        self.axis_of_pair, self.inv_freq = tuple(axis), tuple(freq)
        self.turns = torch.tensor([_turns(f) for f in freq], dtype=torch.int64, device=device)
        self.axis = torch.tensor(axis, dtype=torch.uint8, device=device)

    @property
    def device(self) -> torch.device:
        return self.turns.device

    def to(self, device) -> "RotaryAxes":
        """The same plan with its tables on another device."""
        other = object.__new__(RotaryAxes)
        other.__dict__.update(self.__dict__)
        other.turns, other.axis = self.turns.to(device), self.axis.to(device)
        return other

    def __repr__(self) -> str:
        return f"RotaryAxes({self.head_dim}, {self.sections}, layout={self.layout!r}, device={self.device})"


def _rotary_call(q, k, positions, rotary, q_weight, k_weight, q_bias, k_bias, norm, eps, weight_offset, in_place):
    if not isinstance(rotary, RotaryAxes):
        raise TypeError("rotary must be a RotaryAxes")
    _require_cuda(q, "q")
    if q.dim() < 2 or q.shape[-1] != rotary.head_dim:
        raise RuntimeError(f"q must be [.., heads, {rotary.head_dim}], got {tuple(q.shape)}")
    conf = (rotary.pairs, rotary.axes, _LAYOUTS[rotary.layout], _choice(_KINDS, norm, "norm"), float(eps),
            float(weight_offset), rotary.magnitude)
    args = (q, k, positions, rotary.turns, rotary.axis, q_weight, k_weight, q_bias, k_bias)
    if in_place or not torch.compiler.is_compiling():
        return _ext.qk_norm_rotary(*args, *conf, in_place)
    qo, ko = _t.qk_norm_rotary_fwd(*args, *conf)
    return qo, (ko if k is not None else None)


def fused_qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryAxes,
                         q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                         q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, *,
                         norm: Optional[str] = "rmsnorm", eps: float = 1e-6,
                         weight_offset: float = 0.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q', k'): every head of q [.., q_heads, head_dim] and k [.., k_heads, head_dim] normalized
    over its head_dim elements ("rmsnorm", "layernorm" or "none"; scaled by (weight_offset +
    weight) and shifted by bias, both [head_dim]), then turned by its token's positions as
    `rotary` says.  One launch; q' and k' are contiguous.  k may be None.

    q and k agree in all dimensions but the number of heads, which may differ (grouped heads), and
    may be views of one packed projection or transposed: strides are taken as they are, as long
    as the last dimension is contiguous and the leading ones fold into (batch, sequence).
    positions: int32 or int64, [axes, *tokens] where tokens are the leading dimensions of q, or
    [axes, sequence] for all of the batch, without the axes where there is one.  head_dim <= 512.
    Differentiable in q, k, weights and biases; nothing but the inputs is kept for the backward."""
    return _rotary_call(q, k, positions, rotary, q_weight, k_weight, q_bias, k_bias, norm, eps, weight_offset, False)


def fused_qk_norm_rotary_(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryAxes,
                          q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                          q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, *,
                          norm: Optional[str] = "rmsnorm", eps: float = 1e-6,
                          weight_offset: float = 0.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """fused_qk_norm_rotary written over q and k (returned): for serving, where the heads stay
    inside the packed projection.  Records no gradient (call it under torch.no_grad() when q, k or a
    parameter requires one) and needs strides that it can take as they are; q and k must not overlap."""
    return _rotary_call(q, k, positions, rotary, q_weight, k_weight, q_bias, k_bias, norm, eps, weight_offset, True)


class FusedQKNormRotary(nn.Module):
    """fused_qk_norm_rotary with its parameters: q_weight and k_weight of [head_dim], and with
    bias=True (layer norms) q_bias and k_bias.

        q, k = m(q, k, positions)          # m.forward_(q, k, positions): in place, for serving
    The plan's tables follow the module to another device."""

    def __init__(self, rotary: RotaryAxes, norm: Optional[str] = "rmsnorm", bias: bool = False, eps: float = 1e-6,
                 weight_offset: float = 0.0, elementwise_affine: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        self.norm, self.eps, self.weight_offset = norm or "none", eps, weight_offset
        _choice(_KINDS, self.norm, "norm")
        self._rotary = rotary
        affine = self.norm != "none" and elementwise_affine
        for name, present, value in (("q_weight", affine, 1.0 - weight_offset), ("k_weight", affine, 1.0 - weight_offset),
                                     ("q_bias", affine and bias, 0.0), ("k_bias", affine and bias, 0.0)):
            self.register_parameter(name, Parameter(torch.full((rotary.head_dim,), value, device=device, dtype=dtype))
                                    if present else None)

    @property
    def rotary(self) -> RotaryAxes:
        return self._rotary

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        device = fn(torch.empty(0, device=self._rotary.device)).device
        if device != self._rotary.device:
            self._rotary = self._rotary.to(device)
        return self

    def forward(self, q, k, positions):
        return fused_qk_norm_rotary(q, k, positions, self._rotary, self.q_weight, self.k_weight, self.q_bias, self.k_bias,
                                    norm=self.norm, eps=self.eps, weight_offset=self.weight_offset)

    def forward_(self, q, k, positions):
        return fused_qk_norm_rotary_(q, k, positions, self._rotary, self.q_weight, self.k_weight, self.q_bias, self.k_bias,
                                     norm=self.norm, eps=self.eps, weight_offset=self.weight_offset)

    def extra_repr(self) -> str:
        return f"{self._rotary!r}, norm={self.norm!r}, eps={self.eps}"
