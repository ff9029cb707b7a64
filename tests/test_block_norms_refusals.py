"""Calls of the block norms that are refused before anything is launched: no GPU needed."""
import pytest
import torch
import torch.autograd.forward_ad as fwd_ad

import fused_layernorm as fl
import fused_layernorm_cuda as ext

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
