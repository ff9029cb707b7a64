"""The block-norm operators in 64 bits (plain torch, differentiated by torch), and the error that
a 32-bit evaluation with rounded inputs and outputs may have, propagated to first order.

Bounds.  u is half a step of the tensors' type relative to the value; e24 = E * 2**-24 covers the
32-bit arithmetic of one quantity, E = 48 + n / 64 roundings: a row sum of n terms over at least
64 lanes or accumulators adds n / 64 serial roundings, and some 48 cover the tree, the handful of
elementwise operations and (at 16-bit types) the hardware exponential, reciprocal and reciprocal
square root, each of which is good to 2**-21.  Errors of inputs of an operation are propagated
with absolute values, so the bounds hold for any signs.
"""
import torch

EPS1, EPS2 = 1e-6, 1e-5


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def act_of(v, act):
    if act == "sigmoid":
        return torch.sigmoid(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "tanh":
        return torch.tanh(v)
    return v


def act_grad(v, act):
    if act == "sigmoid":
        q = torch.sigmoid(v)
        return q * (1 - q)
    if act == "silu":
        q = torch.sigmoid(v)
        return q * (1 + v * (1 - q))
    if act == "tanh":
        return 1 - torch.tanh(v) ** 2
    return torch.ones_like(v)


def norm_of(z, kind, w, b, off, eps):
    """(value, xhat, rstd, mean, factor)"""
    mean = z.mean(-1, keepdim=True) if kind == "layernorm" else torch.zeros_like(z[..., :1])
    if kind == "none":
        rstd, xh = torch.ones_like(mean), z
    else:
        rstd = 1 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + eps)
        xh = (z - mean) * rstd
    f = torch.ones_like(z[..., :1]) if w is None else w + off
    n = xh * f
    return (n if b is None else n + b), xh, rstd, mean, f


def spread(t, x):
    """[hidden], [batch, .., hidden] or the shape of x, made to broadcast against x."""
    if t is None or t.dim() == 1 or t.shape == x.shape:
        return t
    return t.reshape(t.shape[0], *([1] * (x.dim() - 2)), t.shape[-1])


def nga_formula(x, residual, gate, w1, b1, w2, b2, post, norm, act, ba, ra, off):
    n1, *_ = norm_of(x, post, w1, b1, off, EPS1)
    a = 1.0 if gate is None else act_of(spread(gate, x), act)
    s = ba * a * n1
    if residual is not None:
        s = s + ra * residual
    y = norm_of(s, norm, spread(w2, x), spread(b2, x), off, EPS2)[0]
    return (None if norm == "none" else y), s


NAMES = ("input", "residual", "gate", "post_weight", "post_bias", "weight", "bias")


def nga_bounds(t, dy, ds, dtype, post, norm, act, ba, ra, off):
    """Values and error bounds of (y, sum) and, with ds, of the seven gradients; t: float64
    tensors by name."""
    x = t["input"]
    h = x.shape[-1]
    u, e24 = u_of(dtype), (48 + h / 64) * 2.0 ** -24
    gate, w1, b1 = spread(t["gate"], x), t["post_weight"], t["post_bias"]
    w2, b2 = spread(t["weight"], x), spread(t["bias"], x)
    n1, xh, r1, m1, f1 = norm_of(x, post, w1, b1, off, EPS1)
    a = torch.ones_like(x[..., :1]) if gate is None else act_of(gate, act)
    s = ba * a * n1 + (0 if t["residual"] is None else ra * t["residual"])
    y, sh, r2, m2, f2 = norm_of(s, norm, w2, b2, off, EPS2)
    mean_abs = x.abs().mean(-1, keepdim=True) if post == "layernorm" else 0.0
    dxh = e24 * (r1 * (x.abs() + mean_abs) + xh.abs())
    dn1 = f1.abs() * dxh + e24 * (xh.abs() * ((0 if w1 is None else w1.abs()) + abs(off)) + (0 if b1 is None else b1.abs()))
    gate_e = e24 * (1 if gate is None else 1 + gate.abs())  # the exponential's argument rounds too
    dlt_s = abs(ba) * (a.abs() * dn1 + gate_e * (a.abs() + (0 if gate is None else 2.0 ** -20)) * n1.abs()) + e24 * (
        (ba * a * n1).abs() + (0 if t["residual"] is None else (ra * t["residual"]).abs()))
    out = {"sum": (s, u * s.abs() + dlt_s)}

    def stat_error(d):  # of xhat of the second norm from an elementwise error d of s
        rms = torch.sqrt((d ** 2).mean(-1, keepdim=True)) if norm != "none" else 0.0
        md = d.mean(-1, keepdim=True) if norm == "layernorm" else 0.0
        ma = s.abs().mean(-1, keepdim=True) if norm == "layernorm" else 0.0
        return r2 * (d + md + e24 * (s.abs() + ma)) + sh.abs() * (r2 * rms + e24)

    if norm != "none":
        out["y"] = (y, u * y.abs() + f2.abs() * stat_error(dlt_s) + e24 * (
            sh.abs() * ((0 if w2 is None else w2.abs()) + abs(off)) + (0 if b2 is None else b2.abs())))
    if dy is None and ds is None:
        return out

    def down(v, like):
        v = v.expand(x.shape)
        if like.shape == x.shape:
            return v
        if like.dim() == 1:
            return v.reshape(-1, h).sum(0)
        return v.reshape(like.shape[0], -1, h).sum(1).reshape(like.shape)

    rows = x.numel() // h
    s24 = e24 + (64 + rows / 64) * 2.0 ** -24  # sums over rows
    dsv = torch.zeros_like(x) if ds is None else ds
    dlt_ds = e24 * dsv.abs()
    dlt_sh = None
    if dy is not None:
        dlt_sh = stat_error(dlt_s)
        g2 = dy * f2
        c1 = (g2 * sh).mean(-1, keepdim=True)
        c2 = g2.mean(-1, keepdim=True) if norm == "layernorm" else 0.0 * c1
        if norm == "none":
            raise ValueError("dy without a norm")
        dg2 = e24 * dy.abs() * ((0 if w2 is None else w2.abs()) + abs(off) + f2.abs())
        dc1 = (g2.abs() * dlt_sh + dg2 * sh.abs()).mean(-1, keepdim=True) + e24 * (g2 * sh).abs().mean(-1, keepdim=True)
        dc2 = (dg2 + e24 * g2.abs()).mean(-1, keepdim=True) if norm == "layernorm" else 0.0
        term = r2 * ((g2 - c2) - sh * c1)
        dr2 = r2 * (r2 * torch.sqrt((dlt_s ** 2).mean(-1, keepdim=True)) + e24)
        dlt_ds = dlt_ds + r2 * (dg2 + dc2 + sh.abs() * dc1 + c1.abs() * dlt_sh + e24 * (g2.abs() + c2.abs() + (sh * c1).abs())) \
            + dr2 * ((g2 - c2) - sh * c1).abs()
        dsv = dsv + term
    e = ba * dsv
    de = abs(ba) * dlt_ds + e24 * e.abs()
    f = e * a
    df = a.abs() * de + gate_e * (a.abs() + (0 if gate is None else 2.0 ** -20)) * e.abs()
    grads = {}
    if t["residual"] is not None:
        v = ra * dsv
        grads["residual"] = (v, u * v.abs() + abs(ra) * dlt_ds + e24 * v.abs())
    g1 = f * f1
    dg1 = f1.abs() * df + e24 * f.abs() * ((0 if w1 is None else w1.abs()) + abs(off) + f1.abs())
    if post == "none":
        grads["input"] = (g1, u * g1.abs() + dg1)
    else:
        d1 = (g1 * xh).mean(-1, keepdim=True)
        d2 = g1.mean(-1, keepdim=True) if post == "layernorm" else 0.0 * d1
        dd1 = (dg1 * xh.abs() + g1.abs() * dxh).mean(-1, keepdim=True) + e24 * (g1 * xh).abs().mean(-1, keepdim=True)
        dd2 = (dg1 + e24 * g1.abs()).mean(-1, keepdim=True) if post == "layernorm" else 0.0
        v = r1 * ((g1 - d2) - xh * d1)
        grads["input"] = (v, u * v.abs() + r1 * (dg1 + dd2 + xh.abs() * dd1 + d1.abs() * dxh + e24 * (
            2 * g1.abs() + 2 * d2.abs() + 3 * (xh * d1).abs())))
    if gate is not None:
        da = act_grad(gate, act)
        v = e * n1 * da
        # act' cancels: silu' = q + q v (1 - q) and 1 - q have terms of order one, q is good to
        # 2**-21 at worst (16-bit types) and each of the last operations to 2**-24, so act' is
        # good to 16 * 2**-24 absolutely where it is small, however small it is
        cancel = 16 * 2.0 ** -24
        d = n1.abs() * (da.abs() * de + (gate_e * da.abs() + cancel) * e.abs()) + (e * da).abs() * dn1
        if gate.shape == x.shape:
            grads["gate"] = tuple(q.reshape(t["gate"].shape) for q in (v, u * v.abs() + d + e24 * v.abs()))
        else:  # act'(gate) * (w1 * sum e xhat + b1 * sum e)
            size = (e * da).abs() * ((xh * f1).abs() + (0 if b1 is None else b1.abs()))
            tot = down(v, t["gate"])
            grads["gate"] = (tot, u * tot.abs() + down(d + s24 * size, t["gate"]))
    if w1 is not None:
        tot = down(f * xh, w1)
        grads["post_weight"] = (tot, u * tot.abs() + down(df * xh.abs() + f.abs() * dxh + s24 * (f * xh).abs(), w1))
    if b1 is not None:
        tot = down(f, b1)
        grads["post_bias"] = (tot, u * tot.abs() + down(df + s24 * f.abs(), b1))
    if dy is not None and w2 is not None:
        tot = down(dy * sh, t["weight"])
        grads["weight"] = (tot, u * tot.abs() + down(dy.abs() * dlt_sh + s24 * (dy * sh).abs(), t["weight"]))
    if dy is not None and b2 is not None:
        tot = down(dy, t["bias"])
        grads["bias"] = (tot, u * tot.abs() + down(s24 * dy.abs(), t["bias"]))
    out["grads"] = grads
    return out


def check(got, bound, what):
    want, tol = bound
    tol = tol.expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what
    tiny = torch.finfo(got.dtype).tiny * 2.0 ** -8 if got.dtype == torch.float16 else 0.0  # fp16 subnormal step
    err = (got.double() - want).abs()
    bad = err > tol + tiny + 1e-30
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {err.numel()} beyond the bound, worst ratio " \
                                f"{(err / (tol + tiny + 1e-30)).max().item():.3g}, error {err.max().item():.3g}"


# ------------------------------------------------------------------------------------ rotary
def rotary_formula(z, pos, axis, inv_freq, layout, kind, w, b, off, eps, mag):
    """pos [axes, *tokens]; returns the rotated rows and what the bounds need."""
    pairs = len(axis)
    n, xh, rstd, mean, f = norm_of(z, kind, w, b, off, eps)
    ang = torch.stack([pos[a].double() * v for a, v in zip(axis, inv_freq)], -1) if pairs else z.new_zeros(*z.shape[:-2], 0)
    c, s = (mag * torch.cos(ang)).unsqueeze(-2), (mag * torch.sin(ang)).unsqueeze(-2)
    i = torch.arange(pairs, device=z.device)
    lo, hi = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    a_, b_ = n[..., lo], n[..., hi]
    ra, rb = a_ * c - b_ * s, b_ * c + a_ * s
    parts = torch.cat([ra, rb, n[..., 2 * pairs:]], -1)
    order = torch.cat([lo, hi, torch.arange(2 * pairs, z.shape[-1], device=z.device)])
    return parts[..., torch.argsort(order)], n, xh, rstd, f, lo, hi
