"""What the block-norm operators refuse and plan on the host, without a GPU: argument errors of
the C entry points, the rotary plan, names, schemas and fake tensors."""
import ctypes as C
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fused_layernorm as fl
from fused_layernorm import _capi as capi

L = capi.lib()


def nga(**kw):
    a = capi.NgaArgs(rows=4, cols=8, group_rows=4, dtype=0, post_kind=1, kind=1, branch_scale=1, residual_scale=1, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_norm_gate_add_norm_argument_errors():
    fwd = lambda a: L.fln_norm_gate_add_norm_forward(C.byref(a), *[None] * 7)
    assert L.fln_norm_gate_add_norm_forward(None, *[None] * 7) == 3
    for kw, st in ((dict(dtype=3), 1), (dict(cols=0), 2), (dict(rows=-1), 2), (dict(group_rows=3), 2), (dict(group_rows=0), 2),
                   (dict(kind=3), 8), (dict(post_kind=-1), 8), (dict(gate_mode=4), 8), (dict(gate_act=4), 8),
                   (dict(gate_mode=1), 8), (dict(gate=64), 8), (dict(kind=2, weight=64), 8), (dict(post_kind=2, post_bias=64), 8),
                   (dict(), 3)):
        assert fwd(nga(**kw)) == st, kw
    assert fwd(nga(rows=0)) == 0
    # outputs may not be inputs
    for y, total in ((64, 128), (128, 64), (128, 128)):
        a = nga(x=64, residual=64)
        assert L.fln_norm_gate_add_norm_forward(C.byref(a), y, total, *[None] * 5) == 8
    bwd = lambda a, p, n=0: L.fln_norm_gate_add_norm_backward(C.byref(a), *p, n, None)
    none = [None] * 14
    assert bwd(nga(), none) == 3  # no gradient arrives
    assert bwd(nga(), none[:8] + [64] + none[9:]) == 8  # dgate without a gate
    assert bwd(nga(x=64), [64] * 6 + [None] * 5 + [64] + [None] * 2) == 4  # dweight without scratch
    assert bwd(nga(x=64), [64] * 6 + [64] + [None] * 7) == 8  # dx over x
    assert L.fln_norm_gate_add_norm_workspace_bytes(C.byref(nga(kind=7))) == 0
    assert L.fln_norm_gate_add_norm_workspace_bytes(C.byref(nga())) > 0


def rot(**kw):
    a = capi.RotaryArgs(batch=1, seq=4, head_dim=64, pairs=32, dtype=0, kind=1, eps=1e-6, magnitude=1)
    a.t[0].heads = 2
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_qk_norm_rotary_argument_errors():
    fwd = lambda a: L.fln_qk_norm_rotary_forward(C.byref(a), None)
    assert L.fln_qk_norm_rotary_forward(None, None) == 3
    for kw, st in ((dict(dtype=9), 1), (dict(head_dim=0), 2), (dict(pairs=33), 2), (dict(pairs=-1), 2), (dict(batch=-1), 2),
                   (dict(seq=1 << 31), 2), (dict(batch=1 << 20, seq=1 << 20), 2), (dict(head_dim=513), 6), (dict(kind=5), 8),
                   (dict(layout=2), 8), (dict(), 3)):
        assert fwd(rot(**kw)) == st, kw
    a = rot(kind=2)
    a.t[0].weight = 64
    assert fwd(a) == 8
    assert fwd(rot(seq=0)) == 0
    pair = C.c_void_p * 2
    a = rot(positions=64, turns=64, axis=64)
    a.t[0].in_ = a.t[0].out = 64
    bwd = lambda a, *g: L.fln_qk_norm_rotary_backward(C.byref(a), *g, None, 0, None)
    assert bwd(a, pair(), pair(64), pair()) == 4  # weight gradient without scratch
    assert bwd(rot(kind=2), pair(), pair(64), pair()) == 8
    assert bwd(rot(), pair(), pair(), pair()) == 3
    assert L.fln_qk_norm_rotary_workspace_bytes(C.byref(rot())) > 0
    assert L.fln_qk_norm_rotary_workspace_bytes(C.byref(rot(head_dim=513))) == 0


def test_rotary_plan():
    r = fl.RotaryAxes(128, (16, 24, 24), base=1e6, device="cpu")
    assert r.axes == 3 and r.pairs == 64 and r.axis_of_pair == (0,) * 16 + (1,) * 24 + (2,) * 24
    assert all(math.isclose(f, 1e6 ** (-i / 64), rel_tol=1e-15) for i, f in enumerate(r.inv_freq))
    p = fl.RotaryAxes(72, (4, 6), per_axis=True, layout="interleaved", device="cpu")
    assert p.inv_freq[:4] == tuple(1e4 ** (-i / 4) for i in range(4)) and p.inv_freq[4:] == tuple(1e4 ** (-i / 6) for i in range(6))
    d = fl.RotaryAxes(16, (2, 4, 1), interleaved_axes=True, device="cpu")
    assert d.axis_of_pair == (0, 1, 2, 0, 1, 1, 1)
    s = fl.RotaryAxes(8, (2, 2), position_scale=(1.0, 0.5), inv_freq=[1.0, 0.5, 0.25, 0.125], device="cpu")
    assert s.inv_freq == (1.0, 0.5, 0.125, 0.0625)
    # turns: inv_freq / 2 pi as a fraction of 2**64, to the last bit that a double can tell
    for f, t in zip(r.inv_freq, r.turns.tolist()):
        assert abs((t % 2 ** 64) / 2 ** 64 - f / (2 * math.pi)) <= 2.0 ** -53
    assert r.turns.dtype == torch.int64 and r.axis.dtype == torch.uint8 and r.to("cpu").axis_of_pair == r.axis_of_pair
    for bad in (lambda: fl.RotaryAxes(64, 33, device="cpu"), lambda: fl.RotaryAxes(64, (-1, 3), device="cpu"),
                lambda: fl.RotaryAxes(64, (), device="cpu"), lambda: fl.RotaryAxes(64, 32, layout="other", device="cpu"),
                lambda: fl.RotaryAxes(64, 32, base=0.0, device="cpu"), lambda: fl.RotaryAxes(64, 2, inv_freq=[1.0], device="cpu"),
                lambda: fl.RotaryAxes(64, 2, inv_freq=[1.0, float("inf")], device="cpu"),
                lambda: fl.RotaryAxes(64, (1, 1), position_scale=(1.0,), device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_names_and_cpu_tensors():
    for n in ("fused_norm_gate_add_norm", "FusedNormGateAddNorm", "RotaryAxes", "fused_qk_norm_rotary", "fused_qk_norm_rotary_",
              "FusedQKNormRotary"):
        assert n in fl.__all__ and hasattr(fl, n)
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        fl.fused_norm_gate_add_norm(x)
    plan = fl.RotaryAxes(8, 4, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        fl.fused_qk_norm_rotary(torch.zeros(2, 1, 8), None, torch.zeros(2, dtype=torch.int64), plan)
    for kw in (dict(post_norm="batch"), dict(norm=1), dict(gate_activation="gelu")):
        with pytest.raises(ValueError):
            fl.fused_norm_gate_add_norm(x, **kw)
    with pytest.raises(TypeError):
        fl.fused_qk_norm_rotary(torch.zeros(2, 1, 8), None, torch.zeros(2, dtype=torch.int64), None)
    with pytest.raises(ValueError):
        fl.FusedNormGateAddNorm(8, norm="other")
    m = fl.FusedNormGateAddNorm(8, post_norm=None, norm="layernorm", bias=True)
    assert set(m.state_dict()) == {"weight", "bias"}
    q = fl.FusedQKNormRotary(plan, norm="layernorm", bias=True)
    assert set(q.state_dict()) == {"q_weight", "k_weight", "q_bias", "k_bias"} and q.half().q_weight.dtype == torch.float16


def test_fake_tensors():
    o = torch.ops.fused_layernorm
    with FakeTensorMode():
        x = torch.empty(2, 3, 8, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(8, dtype=torch.bfloat16, device="cuda")
        y, s, m1, r1, m2, r2 = o.norm_gate_add_norm_fwd(x, x, None, w, None, w, None, 1, 0, 0, 1.0, 1.0, 0.0, 1e-6, 1e-6)
        assert y.shape == s.shape == x.shape and y.dtype == x.dtype
        assert m1.numel() == 0 and r1.shape == m2.shape == r2.shape == (6,) and r2.dtype == torch.float32
        g = o.norm_gate_add_norm_bwd(x, x, x, x, None, w, None, w, None, m1, r1, m2, r2, 1, 0, 0, 1.0, 1.0, 0.0, 1e-6, 1e-6,
                                     [True, True, False, True, False, False, False])
        assert [tuple(t.shape) for t in g] == [(2, 3, 8), (2, 3, 8), (0,), (8,), (0,), (0,), (0,)]
        q = torch.empty(5, 4, 8, device="cuda")
        pos, t, a = torch.empty(5, dtype=torch.int64, device="cuda"), torch.empty(4, dtype=torch.int64, device="cuda"), \
            torch.empty(4, dtype=torch.uint8, device="cuda")
        qo, ko = o.qk_norm_rotary_fwd(q, None, pos, t, a, None, None, None, None, 4, 1, 0, 2, 1e-6, 0.0, 1.0)
        assert qo.shape == q.shape and ko.numel() == 0
