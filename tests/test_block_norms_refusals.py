"""Calls of the block norms that are refused before anything is launched: no GPU needed."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import fused_layernorm as fl
import fused_layernorm_cuda as ext
from fused_layernorm import _capi as capi

NORM = dict(post_kind=1, kind=1, gate_act=0, branch_scale=1.0, residual_scale=1.0, weight_offset=0.0, post_eps=1e-6, eps=1e-6)
ROTARY = dict(pairs=4, axes=1, layout=0, kind=1, eps=1e-6, weight_offset=0.0, magnitude=1.0)


@pytest.mark.parametrize("name", ["input", "residual", "gate", "post_weight", "post_bias", "weight", "bias"])
@pytest.mark.parametrize("grad", [True, False])
def test_norm_gate_add_norm_refuses_forward_mode(name, grad):
    """A dual tensor made from an ordinary one does not require grad, and forward mode goes on under
    no_grad: both are refused, in whatever tensor the tangent sits."""
    t = dict.fromkeys(["input", "residual", "gate", "post_weight", "post_bias", "weight", "bias"])
    t["input"], t[name] = torch.zeros(2, 8), torch.zeros(*((2, 8) if name in ("input", "residual", "gate") else (8,)))
    with fwd_ad.dual_level(), torch.set_grad_enabled(grad):
        t[name] = fwd_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ext.norm_gate_add_norm(**t, **NORM)


@pytest.mark.parametrize("name", ["q", "k", "q_weight", "k_weight", "q_bias", "k_bias"])
@pytest.mark.parametrize("in_place", [True, False])
def test_qk_norm_rotary_refuses_forward_mode(name, in_place):
    plan = fl.RotaryAxes(8, 4, device="cpu")
    t = dict.fromkeys(["q_weight", "k_weight", "q_bias", "k_bias"])
    t["q"], t["k"] = torch.zeros(3, 2, 8), torch.zeros(3, 1, 8)
    if t.get(name) is None:
        t[name] = torch.zeros(8)
    with fwd_ad.dual_level():
        t[name] = fwd_ad.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ext.qk_norm_rotary(**t, positions=torch.zeros(3, dtype=torch.int64), turns=plan.turns, axis=plan.axis, **ROTARY,
                               in_place=in_place)


# ------------------------------------------------------------------------------ written in place
def elements(t):
    """Storage places of all elements, one by one."""
    at = torch.tensor(t.storage_offset())
    for size, stride in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(size) * stride
    return at.flatten().tolist()


def apart(q, k):
    a, b = elements(q), elements(k)
    return len(set(a)) == len(a) and len(set(b)) == len(b) and not set(a) & set(b)


def refused(q, k):
    try:
        ext.check_rotary_in_place(q, k)
    except RuntimeError:
        return True
    return False


def test_in_place_takes_the_views_of_a_projection():
    """What serving code hands in: views of a packed projection with any number of leading
    dimensions, heads before tokens, separate tensors, k behind or in front of q."""
    for lead in ((6,), (2, 3), (2, 2, 3), (1, 5), (3, 1)):
        p = torch.zeros(*lead, 8, 4)
        for q, k in ((p[..., :5, :], p[..., 5:7, :]), (p[..., 3:, :], p[..., :3, :]), (p[..., :1, :], p[..., 1:2, :]),
                     (p[..., :5, :], torch.zeros(*lead, 2, 4)), (p, None)):
            assert not refused(q, k)
    p = torch.zeros(8, 6, 4)
    assert not refused(p[:5].transpose(0, 1), p[5:7].transpose(0, 1))
    p = torch.zeros(2, 8, 6, 4)
    assert not refused(p[:, :5].transpose(1, 2), p[:, 5:7].transpose(1, 2))


def test_in_place_refuses_elements_in_common():
    """q fits between its own rows but k reaches from one batch entry into the next one's q."""
    s = torch.zeros(64)
    q, k = s.as_strided((2, 3, 1, 4), (20, 8, 4, 1), 0), s.as_strided((2, 3, 1, 4), (20, 8, 4, 1), 4)
    assert not apart(q, k) and apart(q, s.as_strided((1, 1, 1, 4), (1, 1, 4, 1), 60))
    assert refused(q, k) and refused(k, q) and not refused(q, None)


def test_in_place_never_takes_what_is_not_apart():
    """Strided views at random over one small storage, against a list of their elements.  The check
    may refuse what a list would allow, never the other way round."""
    g = torch.Generator().manual_seed(3)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    s = torch.zeros(400)
    taken = shared = 0
    for _ in range(4000):
        b, n, d = r(1, 3), r(1, 3), r(1, 4)
        stride = (r(1, 40), r(1, 20), r(1, 8))
        views = []
        for _ in range(2):
            own = stride if r(0, 3) else (r(1, 40), r(1, 20), r(1, 8))
            views.append(s.as_strided((b, n, r(1, 3), d), (*own, 1), r(0, 40)))
        ok = apart(*views)
        shared += not ok
        if not refused(*views):
            taken += 1
            assert ok, [(v.shape, v.stride(), v.storage_offset()) for v in views]
    assert taken > 100 and shared > 100


# ------------------------------------------------------------------ outputs over inputs, C functions
L = capi.lib()
ROWS, COLS = 4, 64  # fp32: a tensor is 1024 bytes, a vector 256, a statistic 16


def nga_args(**kw):
    a = capi.NgaArgs(rows=ROWS, cols=COLS, group_rows=2, dtype=capi.F32, post_kind=capi.LAYERNORM, kind=capi.LAYERNORM, branch_scale=1,
                     residual_scale=1, eps=1e-6, gate_mode=capi.GATE_ELEMENT, affine_grouped=1)
    at = 1 << 20
    for n in ("x", "residual", "gate", "post_weight", "post_bias", "weight", "bias"):
        setattr(a, n, at)
        at += 1 << 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SIZE = dict(x=1024, residual=1024, gate=1024, post_weight=256, post_bias=256, weight=512, bias=512)


@pytest.mark.parametrize("name", list(SIZE))
@pytest.mark.parametrize("out", ["y", "sum", "post_mean", "post_rstd", "mean", "rstd"])
def test_forward_refuses_outputs_that_reach_into_inputs(name, out):
    """The first and the last place at which an output overlaps a tensor, in whole elements."""
    outs = ["y", "sum", "post_mean", "post_rstd", "mean", "rstd"]
    own = 1024 if out in ("y", "sum") else 16
    a = nga_args()
    base = getattr(a, name)
    for at in (base, base + SIZE[name] - 4, base - own + 4):
        p = [at if o == out else (1 << 24) + (i << 16) for i, o in enumerate(outs)]
        assert L.fln_norm_gate_add_norm_forward(C.byref(a), *p, None) == 8, (name, out, at - base)


def test_forward_refuses_outputs_that_overlap_each_other():
    outs = [(1 << 24) + (i << 16) for i in range(6)]
    size = [1024, 1024, 16, 16, 16, 16]
    for i in range(6):
        for j in range(6):
            if i == j:
                continue
            for at in (outs[j], outs[j] + size[j] - 4):
                p = list(outs)
                p[i] = at
                assert L.fln_norm_gate_add_norm_forward(C.byref(nga_args()), *p, None) == 8


def test_backward_refuses_outputs_that_reach_into_inputs_or_each_other():
    a = nga_args()
    need = L.fln_norm_gate_add_norm_workspace_bytes(C.byref(a))
    ins = dict(SIZE, post_mean=16, post_rstd=16, mean=16, rstd=16, dy=1024, dsum=1024)
    del ins["bias"]  # the one tensor that the backward does not read
    outs = dict(dx=1024, dresidual=1024, dgate=1024, dpost_weight=256, dpost_bias=256, dweight=512, dbias=512)
    at = {n: (1 << 24) + (i << 16) for i, n in enumerate(["post_mean", "post_rstd", "mean", "rstd", "dy", "dsum", *outs])}
    args = list(at)
    where = lambda n: at[n] if n in at else getattr(a, n)

    def call(workspace=1 << 28, **moved):
        return L.fln_norm_gate_add_norm_backward(C.byref(a), *[moved.get(n, at[n]) for n in args], workspace, need, None)

    for o, own in outs.items():
        for n, size in [*ins.items(), *((n, s) for n, s in outs.items() if n != o)]:
            for place in (where(n), where(n) + size - 4, where(n) - own + 4):
                assert call(**{o: place}) == 8, (o, n)
        assert call(workspace=at[o] - need // 16 * 16 + 16) == 8  # the end of the scratch in a gradient
    for n in ins:
        assert call(workspace=where(n) // 16 * 16) == 8, n


def test_rotary_in_place_takes_the_same_strides_only():
    a = capi.RotaryArgs(batch=2, seq=4, head_dim=64, pairs=32, dtype=capi.F32, kind=capi.RMSNORM, eps=1e-6, magnitude=1, positions=64,
                        turns=64, axis=64)
    t = a.t[0]
    t.heads, t.in_, t.out = 2, 1 << 20, 1 << 20
    strides = dict(batch=2048, seq=512, head=128)
    for k, v in strides.items():
        setattr(t, "in_" + k, v), setattr(t, "out_" + k, v)
    for k, v in strides.items():
        setattr(t, "out_" + k, v // 2)
        assert L.fln_qk_norm_rotary_forward(C.byref(a), None) == 8
        setattr(t, "out_" + k, v)
