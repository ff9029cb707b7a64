"""fused_qk_norm_rotary (head norm, then the rotation of multi-axis rotary positions) against the
formula in 64 bits: values, gradients, differences, layouts, strides, in place, refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import block_norms_ref as R

if torch.cuda.is_available():
    import fused_layernorm as fl

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def positions(lead, axes, far=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-50, 5000, (axes, *lead), generator=g).cuda() + far


def make(lead, hq, hk, dim, dtype, norm="rmsnorm", bias=False, affine=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    t = {"q": rn(*lead, hq, dim) * 1.3 + 0.2, "k": rn(*lead, hk, dim) - 0.1 if hk else None}
    has = norm != "none" and affine
    for s in ("q", "k"):
        there = has and t[s] is not None
        t[s + "_weight"] = 1.0 + 0.2 * rn(dim) if there else None
        t[s + "_bias"] = 0.2 * rn(dim) if there and bias else None
    t["dq"], t["dk"] = rn(*lead, hq, dim), rn(*lead, hk, dim) if hk else None
    return {k: None if v is None else v.to(dtype).cuda() for k, v in t.items()}


def call(t, pos, rot, norm, off=0.0, fn=None):
    return (fn or fl.fused_qk_norm_rotary)(t["q"], t["k"], pos, rot, t["q_weight"], t["k_weight"], t["q_bias"], t["k_bias"],
                                           norm=norm, eps=EPS, weight_offset=off)


def full_pos(pos, rot, lead):
    if rot.axes == 1 and (pos.shape == lead or pos.dim() == 1):
        pos = pos[None]
    while pos.dim() < 1 + len(lead):
        pos = pos.unsqueeze(1)
    return pos.expand(rot.axes, *lead)


def bounds(t, pos, rot, norm, off, s):
    """Value, gradients and their bounds for one of the two tensors."""
    z = t[s].detach().double()
    dim = z.shape[-1]
    u, e24 = R.u_of(t[s].dtype), (48 + dim / 64) * 2.0 ** -24
    d = lambda v: None if v is None else v.detach().double()
    w, b = d(t[s + "_weight"]), d(t[s + "_bias"])
    args = (full_pos(pos, rot, z.shape[:-2]), rot.axis_of_pair, rot.inv_freq, rot.layout, norm, w, b, off, EPS, rot.magnitude)
    o, n, xh, rstd, f, lo, hi = R.rotary_formula(z, *args)

    def mixed(v):  # what a rotation makes of elementwise errors: both members of a pair, times the magnitude
        m = v.clone()
        both = abs(rot.magnitude) * (v[..., lo] + v[..., hi])
        m[..., lo], m[..., hi] = both, both
        return m

    ma = z.abs().mean(-1, keepdim=True) if norm == "layernorm" else 0.0
    dxh = e24 * (rstd * (z.abs() + ma) + xh.abs()) if norm != "none" else 0.0 * z
    dn = f.abs() * dxh + e24 * (xh.abs() * ((0 if w is None else w.abs()) + abs(off)) + (0 if b is None else b.abs()))
    # the angle is wrong by position * 2**-65 turns at most, and its cosine and sine by 2**-22
    out = {"value": (o, u * o.abs() + mixed(dn + 2.0 ** -21 * n.abs()))}
    if t["d" + s] is None:
        return out
    zz = z.clone().requires_grad_(True)
    ps = {k: v.clone().requires_grad_(True) for k, v in (("w", w), ("b", b)) if v is not None}
    oo = R.rotary_formula(zz, *args[:5], ps.get("w"), ps.get("b"), *args[7:])[0]
    g = d(t["d" + s])
    grads = torch.autograd.grad(oo, [zz, *ps.values()], g)
    # rotated back
    dnv = torch.autograd.grad(R.rotary_formula(z.clone(), args[0], args[1], args[2], args[3], "none", None,
                                               (bb := torch.zeros_like(z, requires_grad=True)), 0.0, EPS, args[-1])[0], bb, g)[0]
    ddn = mixed(2.0 ** -21 * g.abs())
    g1 = dnv * f
    dg1 = f.abs() * ddn + e24 * dnv.abs() * ((0 if w is None else w.abs()) + abs(off) + f.abs())
    if norm == "none":
        out["dx"] = (grads[0], u * grads[0].abs() + dg1)
    else:
        mean = lambda v: v.mean(-1, keepdim=True)
        d1, d2 = mean(g1 * xh), mean(g1) if norm == "layernorm" else 0.0
        dd1 = mean(dg1 * xh.abs() + g1.abs() * dxh + e24 * (g1 * xh).abs())
        dd2 = mean(dg1 + e24 * g1.abs()) if norm == "layernorm" else 0.0
        out["dx"] = (grads[0], u * grads[0].abs() + rstd * (dg1 + dd2 + xh.abs() * dd1 + d1.abs() * dxh + e24 * (
            2 * g1.abs() + (2 * d2.abs() if norm == "layernorm" else 0.0) + 3 * (xh * d1).abs())))
    rows = z.numel() // dim
    s24 = e24 + (64 + rows / 64) * 2.0 ** -24
    down = lambda v: v.reshape(-1, dim).sum(0)
    for k, gr, term, err in zip(ps, grads[1:], [x for x, p in ((dnv * xh, w), (dnv, b)) if p is not None],
                                [x for x, p in ((ddn * xh.abs() + dnv.abs() * dxh, w), (ddn, b)) if p is not None]):
        out["d" + k] = (gr, u * gr.abs() + down(err + s24 * term.abs()))
    return out


def check_case(t, pos, rot, norm, off=0.0, fn=None):
    qo, ko = call(t, pos, rot, norm, off)
    want = {s: bounds(t, pos, rot, norm, off, s) for s in ("q", "k") if t[s] is not None}
    R.check(qo, want["q"]["value"], "q")
    assert (ko is None) == (t["k"] is None)
    if ko is not None:
        R.check(ko, want["k"]["value"], "k")
    names = [n for n in ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias") if t[n] is not None]
    leaves = {n: t[n].detach().requires_grad_(True) for n in names}
    q2, k2 = call({**t, **leaves}, pos, rot, norm, off)
    assert torch.equal(q2, qo) and (ko is None or torch.equal(k2, ko))
    outs, gs = ([q2], [t["dq"]]) if ko is None else ([q2, k2], [t["dq"], t["dk"]])
    got = torch.autograd.grad(outs, list(leaves.values()), gs, retain_graph=True)
    for n, g in zip(names, got):
        key = "dx" if n in ("q", "k") else "d" + n[2]
        R.check(g, want[n[0]][key], "d" + n)
    for a, b in zip(got, torch.autograd.grad(outs, list(leaves.values()), gs)):
        assert torch.equal(a, b)


CASES = [  # lead, q heads, k heads, head_dim, sections, options
    ((1,), 1, 1, 2, 1, {}), ((3,), 4, 2, 128, (16, 24, 24), {}), ((16,), 32, 8, 128, 64, {}), ((2, 9), 3, 1, 64, (11, 21), {}),
    ((5,), 2, 2, 72, (12, 12, 12), dict(per_axis=True, layout="interleaved")), ((4, 33), 12, 4, 80, 20, {}),
    ((130,), 5, 5, 96, (16, 16, 16), dict(interleaved_axes=True)), ((7,), 2, 1, 50, 25, {}), ((7,), 2, 1, 51, 20, {}),
    ((2, 3, 5), 2, 2, 112, (20, 36), dict(layout="interleaved")), ((9,), 1, 0, 256, 128, {}), ((65,), 6, 3, 192, 50, {}),
    ((5,), 2, 2, 90, 45, dict(layout="interleaved")), ((3,), 2, 1, 512, (100, 100), {}), ((3,), 2, 1, 511, (100, 101), {}),
    ((6,), 3, 2, 33, 0, {}), ((400,), 40, 8, 128, 64, dict(magnitude=1.2)), ((11,), 2, 1, 510, 255, dict(layout="interleaved")),
    ((70,), 16, 16, 40, (6, 7, 7), dict(position_scale=(1.0, 0.5, 0.25))), ((2,), 130, 1, 128, 64, {})]


@pytest.mark.parametrize("i", range(len(CASES)))
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("norm", ["rmsnorm", "layernorm", "none"])
def test_values_and_gradients(i, dtype, norm):
    lead, hq, hk, dim, sections, opts = CASES[i]
    rot = fl.RotaryAxes(dim, sections, base=1e6 if i % 2 else 1e4, **opts)
    t = make(lead, hq, hk, dim, dtype, norm, bias=i % 2 == 0, affine=i % 7 != 3, seed=i)
    off = 1.0 if i % 3 == 0 and norm != "none" else 0.0
    check_case(t, positions(lead, rot.axes, far=(0, 1 << 17, 1 << 20)[i % 3], seed=i), rot, norm, off)


def test_many_tokens():
    rot = fl.RotaryAxes(64, (8, 12, 12))
    check_case(make((20011,), 3, 2, 64, BF16), positions((20011,), 3), rot, "rmsnorm")
    rot = fl.RotaryAxes(128, 64)
    check_case(make((3, 1111), 8, 2, 128, F32, "layernorm", bias=True), positions((3, 1111), 1), rot, "layernorm")


def test_far_positions_are_exact():
    """Angles at positions up to 2**40: the 64-bit formula in whole turns, by integer arithmetic."""
    dim = 64
    rot = fl.RotaryAxes(dim, 32)
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 40, 2 ** 40 + 1, -2 ** 40 + 7], device="cuda")
    q = torch.zeros(len(pos), 1, dim, device="cuda")
    q[..., :32] = 1.0  # rotates to (cos, sin)
    out, _ = fl.fused_qk_norm_rotary(q, None, pos, rot, norm="none")
    turns = [int(v) % 2 ** 64 for v in rot.turns.tolist()]
    for i, p in enumerate(pos.tolist()):
        frac = torch.tensor([((p * f) % 2 ** 64) / 2 ** 64 for f in turns], dtype=torch.float64)
        want = torch.cat([torch.cos(2 * torch.pi * frac), torch.sin(2 * torch.pi * frac)])
        # 2**-24 for the fraction's rounding (times 2 pi), and for sine and cosine
        assert (out[i, 0].cpu().double() - want).abs().max() <= 6.4 * 2.0 ** -24 + 2.0 ** -22
    # int32 positions give the same values
    small = pos[:5]
    assert torch.equal(fl.fused_qk_norm_rotary(q[:5], None, small.int(), rot, norm="none")[0], out[:5])


def test_offsets_beyond_32_bits():
    """Tokens of a packed projection that lie past 2**31 elements, and dx past them."""
    n, hq, hk, dim = 210000, 70, 10, 128  # 90 heads of 128 in a row of the projection: 2.4e9 elements
    rot = fl.RotaryAxes(dim, (16, 24, 24))
    qkv = torch.empty(n, hq + 2 * hk, dim, dtype=BF16, device="cuda").normal_()
    q, k = qkv[:, :hq].detach().requires_grad_(True), qkv[:, hq:hq + hk].detach().requires_grad_(True)
    pos = positions((n,), 3)
    qo, ko = fl.fused_qk_norm_rotary(q, k, pos, rot, eps=EPS)
    dq, dk = torch.empty_like(qo).normal_(), torch.empty_like(ko).normal_()
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [dq, dk])
    for part in (slice(0, 3), slice(n - 3, n)):
        t = {"q": q[part].detach(), "k": k[part].detach(), "dq": dq[part], "dk": dk[part],
             **dict.fromkeys(("q_weight", "k_weight", "q_bias", "k_bias"))}
        for s, o, gr in (("q", qo, gq), ("k", ko, gk)):
            want = bounds(t, pos[:, part], rot, "rmsnorm", 0.0, s)
            R.check(o[part], want["value"], s), R.check(gr[part], want["dx"], "d" + s)


def test_position_shapes():
    t = make((3, 10), 2, 1, 64, F32)
    one, three = fl.RotaryAxes(64, 32), fl.RotaryAxes(64, (8, 12, 12))
    p = positions((3, 10), 3)
    for rot, pos in ((one, p[0]), (one, p[:1]), (one, p[0, 0]), (one, p[:1, 0]), (three, p), (three, p[:, 0]),
                     (three, p.transpose(1, 2).contiguous().transpose(1, 2)), (three, p.int())):
        check_case(t, pos, rot, "rmsnorm")


def test_views_of_a_packed_projection_and_transposed_heads():
    """q and k as views of one projection, heads first in memory, an unaligned offset; gradients
    that arrive transposed."""
    lead, hq, hk, dim = (4, 37), 6, 2, 96
    t = make(lead, hq, hk, dim, BF16)
    rot = fl.RotaryAxes(dim, (16, 16, 16))
    pos = positions(lead, 3)
    qkv = torch.randn(*lead, hq + 2 * hk, dim, device="cuda").to(BF16)
    qkv[..., :hq, :], qkv[..., hq:hq + hk, :] = t["q"], t["k"]
    check_case({**t, "q": qkv[..., :hq, :], "k": qkv[..., hq:hq + hk, :]}, pos, rot, "rmsnorm")
    hf = lambda v: v.transpose(1, 2).contiguous().transpose(1, 2)
    check_case({**t, "q": hf(t["q"]), "k": hf(t["k"]), "dq": hf(t["dq"]), "dk": hf(t["dk"])}, pos, rot, "rmsnorm")
    odd = torch.zeros(t["q"].numel() + 1, dtype=BF16, device="cuda")
    odd[1:] = t["q"].reshape(-1)
    check_case({**t, "q": odd[1:].view(t["q"].shape)}, pos, rot, "rmsnorm")
    step = torch.zeros(*lead, hq, dim, 2, dtype=BF16, device="cuda")
    step[..., 0] = t["q"]
    check_case({**t, "q": step[..., 0]}, pos, rot, "rmsnorm")
    check_case({**t, "q": t["q"][:, :1].expand(lead[0], lead[1], hq, dim)}, pos, rot, "rmsnorm")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [1, 3, 64, 500])
def test_in_place_inside_a_packed_projection(dtype, tokens):
    hq, hk, dim = 8, 2, 128
    t = make((tokens,), hq, hk, dim, dtype)
    rot = fl.RotaryAxes(dim, 64)
    pos = positions((tokens,), 1)[0]
    qkv = torch.randn(tokens, hq + 2 * hk, dim, device="cuda").to(dtype)
    qkv[:, :hq], qkv[:, hq:hq + hk] = t["q"], t["k"]
    want = call(t, pos, rot, "rmsnorm")
    v = qkv[:, hq + hk:].clone()
    ver = qkv._version
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    got = call({**t, "q": q, "k": k}, pos, rot, "rmsnorm", fn=fl.fused_qk_norm_rotary_)
    assert got[0].data_ptr() == q.data_ptr() and got[1].data_ptr() == k.data_ptr() and qkv._version > ver
    assert torch.equal(qkv[:, :hq], want[0]) and torch.equal(qkv[:, hq:hq + hk], want[1])
    assert torch.equal(qkv[:, hq + hk:], v)
    # heads in front of tokens
    qkv = torch.randn(hq + 2 * hk, tokens, dim, device="cuda").to(dtype)
    qkv[:hq], qkv[hq:hq + hk] = t["q"].transpose(0, 1), t["k"].transpose(0, 1)
    call({**t, "q": qkv[:hq].transpose(0, 1), "k": qkv[hq:hq + hk].transpose(0, 1)}, pos, rot, "rmsnorm",
         fn=fl.fused_qk_norm_rotary_)
    assert torch.equal(qkv[:hq].transpose(0, 1), want[0]) and torch.equal(qkv[hq:hq + hk].transpose(0, 1), want[1])


def test_gradients_against_differences():
    t = make((7,), 3, 2, 48, F32, "layernorm", bias=True, seed=2)
    rot = fl.RotaryAxes(48, (6, 7, 7), layout="interleaved")
    pos = positions((7,), 3)
    names = ["q", "k", "q_weight", "k_weight", "q_bias", "k_bias"]
    leaves = {n: t[n].detach().requires_grad_(True) for n in names}
    qo, ko = call({**t, **leaves}, pos, rot, "layernorm")
    grads = dict(zip(names, torch.autograd.grad([qo, ko], list(leaves.values()), [t["dq"], t["dk"]])))
    loss = lambda o: (o[0].double() * t["dq"].double()).sum() + (o[1].double() * t["dk"].double()).sum()

    def exact(v):
        return loss([R.rotary_formula(v[s].double(), pos, rot.axis_of_pair, rot.inv_freq, rot.layout, "layernorm",
                                      v[s + "_weight"].double(), v[s + "_bias"].double(), 0.0, EPS, 1.0)[0] for s in "qk"])

    ex = {n: v.detach().double().requires_grad_(True) for n, v in leaves.items()}
    slope = dict(zip(names, torch.autograd.grad(exact(ex), list(ex.values()))))
    h = 2.0 ** -7
    g = torch.Generator().manual_seed(9)
    for n in names:
        d = torch.randn(leaves[n].shape, generator=g).cuda()
        vals, exs = [], []
        for sign in (1, -1):
            moved = {m: (v.detach() + sign * h * d if m == n else v.detach()) for m, v in leaves.items()}
            vals.append(loss(call({**t, **moved}, pos, rot, "layernorm")))
            exs.append(exact(moved))
        got, trunc = (vals[0] - vals[1]) / (2 * h), (exs[0] - exs[1]) / (2 * h) - (slope[n] * d.double()).sum()
        noise = 2.0 ** -24 * 60 * ((qo * t["dq"]).double().abs().sum() + (ko * t["dk"]).double().abs().sum()) / h
        assert (got - (grads[n].double() * d.double()).sum()).abs() <= noise + 1.01 * trunc.abs(), n


def test_gradient_of_one_output_alone_and_some_gradients():
    t = make((19,), 4, 2, 64, BF16)
    rot, pos = fl.RotaryAxes(64, 32), positions((19,), 1)
    for s in ("q", "k"):
        v = {n: t[n].detach().requires_grad_(True) for n in ("q", "k", "q_weight", "k_weight")}
        out = call({**t, **v}, pos, rot, "rmsnorm")
        out["qk".index(s)].backward(t["d" + s])
        b = bounds(t, pos, rot, "rmsnorm", 0.0, s)
        R.check(v[s].grad, b["dx"], s)
        R.check(v[s + "_weight"].grad, b["dw"], s)
        other = "k" if s == "q" else "q"
        assert v[other].grad is None or not bool(v[other].grad.any())
    w = t["q_weight"].detach().requires_grad_(True)
    out = call({**t, "q_weight": w}, pos, rot, "rmsnorm")
    R.check(torch.autograd.grad(out[0], w, t["dq"])[0], bounds(t, pos, rot, "rmsnorm", 0.0, "q")["dw"], "dq_weight")


def test_empty():
    rot = fl.RotaryAxes(64, 32)
    for lead in ((0,), (3, 0), (0, 4)):
        t = make(lead, 2, 1, 64, BF16)
        v = {n: t[n].detach().requires_grad_(True) for n in ("q", "k", "q_weight", "k_weight")}
        q, k = call({**t, **v}, positions(lead, 1), rot, "rmsnorm")
        assert q.shape == t["q"].shape and k.shape == t["k"].shape
        (q.sum() + k.sum()).backward()
        assert not bool(v["q_weight"].grad.any()) and not bool(v["k_weight"].grad.any())


def test_graph_capture_and_streams():
    rot, pos = fl.RotaryAxes(128, (16, 24, 24)), positions((50,), 3)
    t = make((50,), 8, 2, 128, BF16)
    leaves = {n: t[n].detach().clone().requires_grad_(True) for n in ("q", "k", "q_weight", "k_weight")}

    def step():
        o = call({**t, **leaves}, pos, rot, "rmsnorm")
        return o + torch.autograd.grad(list(o), list(leaves.values()), [t["dq"], t["dk"]])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            leaves["q"].mul_(0.9).add_(0.1)
            pos.add_(17)
        g.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_refusals():
    rot, pos = fl.RotaryAxes(64, 32), positions((5,), 1)[0]
    t = make((5,), 4, 2, 64, BF16)
    call(t, pos, rot, "rmsnorm")
    bad = [({"k": t["k"][:4]}, pos), ({"k": t["k"].float()}, pos), ({"q_weight": t["q_weight"][:63]}, pos),
           ({"q_weight": t["q_weight"].cpu()}, pos), ({}, pos[:4]), ({}, pos.float()), ({}, pos.cpu()), ({"k": None}, pos),
           ({"q": t["q"][..., :62]}, pos), ({"q": t["q"].cpu()}, pos), ({}, torch.stack([pos, pos]))]
    for change, p in bad:
        with pytest.raises(RuntimeError):
            call({**t, **change}, p, rot, "rmsnorm")
    with pytest.raises(RuntimeError):
        call(t, pos, rot, "none")  # weights without a norm
    with pytest.raises(NotImplementedError):
        fl.fused_qk_norm_rotary(t["q"].double(), None, pos, rot, norm="none")
    with pytest.raises(RuntimeError, match="512"):
        fl.fused_qk_norm_rotary(torch.zeros(2, 1, 520, device="cuda"), None, pos[:2], fl.RotaryAxes(520, 20), norm="none")
    with pytest.raises(RuntimeError, match="same device"):
        call(t, pos, fl.RotaryAxes(64, 32, device="cpu"), "rmsnorm")
    # in place
    inplace = lambda q, k: fl.fused_qk_norm_rotary_(q, k, pos, rot, norm="none")
    both = torch.zeros(5, 8, 64, dtype=BF16, device="cuda")
    inplace(both[:, :4], both[:, 4:6])
    for q, k in ((both[:, :4], both[:, 3:5]), (both[:, :4], both[:, :4]), (both[:, 2:6], both[:, :3]),
                 (both[:1].expand(5, 8, 64), None), (torch.zeros(5, 4, 128, dtype=BF16, device="cuda")[..., ::2], None)):
        with pytest.raises(RuntimeError):
            inplace(q, k)
    with pytest.raises(RuntimeError, match="no gradient"):
        fl.fused_qk_norm_rotary_(t["q"].detach().requires_grad_(True), None, pos, rot, norm="none")
    x = t["q"].detach().requires_grad_(True)
    out, _ = fl.fused_qk_norm_rotary(x, None, pos, rot)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), x, create_graph=True)


def test_module_compile_and_a_whole_block():
    """The operators as a block uses them: norm -> projections -> head norm + rotary, then the
    attention's output through post norm, gate and residual into the next norm; gradients of the
    whole against the plain composition in 64 bits."""
    torch.manual_seed(1)
    h, hq, hk, dim, b, n = 192, 6, 2, 32, 2, 24
    rot = fl.RotaryAxes(dim, (4, 6, 6))
    qkn = fl.FusedQKNormRotary(rot, device="cuda")
    blk = fl.FusedNormGateAddNorm(h, layer_scale=0.3, device="cuda")
    pre = fl.FusedRMSNorm(h, eps=1e-6, device="cuda")
    wqkv = torch.randn(h, (hq + 2 * hk) * dim, device="cuda") * h ** -0.5
    wo = torch.randn(hq * dim, h, device="cuda") * h ** -0.5
    for p in [*qkn.parameters(), *blk.parameters(), *pre.parameters()]:
        p.data.add_(0.1 * torch.randn_like(p))
    pos = positions((b, n), 3)
    x0 = torch.randn(b, n, h, device="cuda")

    def attend(q, k, v):
        k, v = (t.repeat_interleave(hq // hk, 2) for t in (k, v))
        a = torch.einsum("bihd,bjhd->bhij", q, k) * dim ** -0.5
        a = torch.softmax(a.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), float("-inf")), -1)
        return torch.einsum("bhij,bjhd->bihd", a, v).reshape(b, n, -1)

    def ours(x):
        qkv = (pre(x) @ wqkv).view(b, n, hq + 2 * hk, dim)
        q, k = qkn(qkv[:, :, :hq], qkv[:, :, hq:hq + hk], pos)
        return blk(attend(q, k, qkv[:, :, hq + hk:]) @ wo, x)

    params = [*pre.parameters(), *qkn.parameters(), *blk.parameters()]
    x = x0.clone().requires_grad_(True)
    y, s = ours(x)
    got = torch.autograd.grad([y.sum() + (s * s).sum()], [x, *params])
    P = [p.detach().double().requires_grad_(True) for p in params]
    xd = x0.double().requires_grad_(True)
    pw, qw, kw, w1, w2, gate = P
    qkv = (R.norm_of(xd, "rmsnorm", pw, None, 0.0, 1e-6)[0] @ wqkv.double()).view(b, n, hq + 2 * hk, dim)
    q, k = (R.rotary_formula(z, pos, rot.axis_of_pair, rot.inv_freq, "half", "rmsnorm", w, None, 0.0, 1e-6, 1.0)[0]
            for z, w in ((qkv[:, :, :hq], qw), (qkv[:, :, hq:hq + hk], kw)))
    o = attend(q, k, qkv[:, :, hq + hk:]) @ wo.double()
    sd = xd + gate * R.norm_of(o, "rmsnorm", w1, None, 0.0, 1e-6)[0]
    yd = R.norm_of(sd, "rmsnorm", w2, None, 0.0, 1e-6)[0]
    want = torch.autograd.grad([yd.sum() + (sd * sd).sum()], [xd, *P])
    # two products of some 200 fp32 terms (2**-24 * 200, and TF32 is off), amplified by the norms
    for a, w in zip([y, s, *got], [yd, sd, *want]):
        assert (a.double() - w).norm() <= 2e-4 * w.norm() + 1e-6
    assert set(qkn.state_dict()) == {"q_weight", "k_weight"}
    fn = torch.compile(lambda a, c: qkn(a, c, pos), fullgraph=True, backend="aot_eager")
    q0, k0 = torch.randn(b, n, hq, dim, device="cuda", requires_grad=True), torch.randn(b, n, hk, dim, device="cuda")
    e, c = qkn(q0, k0, pos), fn(q0, k0)
    assert torch.equal(e[0], c[0]) and torch.equal(e[1], c[1])
    ge, gc = (torch.autograd.grad(v[0].sum(), [q0, qkn.q_weight]) for v in (e, c))
    assert all(torch.equal(a, d) for a, d in zip(ge, gc))
