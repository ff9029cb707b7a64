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
