"""Cases, plain forms and exact values of the block-norm operators.

Two families:

  norms    fused_norm_gate_add_norm: the norm after a block, its gate and scale, the residual
           add, and the norm in front of the next block.
               s = residual_scale * residual + branch_scale * act(gate) * N1(x);   y = N2(s)
  rotary   fused_qk_norm_rotary: the norm of every q and k head followed by the rotation of
           rotary positions with one or several axes (time, height, width).

`run` computes one pass of a case: a forward call, or a training step (forward and backward
through autograd, gradients returned).  With `own` false it uses elementary torch operations in
32 bits (angles in 64), rounded once at the end.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "fused-layernorm-cuda-operator_b200")
_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _fl():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import fused_layernorm
    return fused_layernorm


# ------------------------------------------------------------------------------------- cases
def _norms(name, batch, tokens, hidden, dtype, step=False, post="rmsnorm", norm="rmsnorm", gate="none", act="none",
           affine="vector", bias=False, residual=True, branch_scale=1.0, residual_scale=1.0, offset=0.0):
    return {"name": name, "op": "norms", "batch": batch, "tokens": tokens, "hidden": hidden, "dtype": dtype, "step": step,
            "post": post, "norm": norm, "gate": gate, "act": act, "affine": affine, "bias": bias, "residual": residual,
            "branch_scale": branch_scale, "residual_scale": residual_scale, "offset": offset}


def _rotary(name, tokens, q_heads, k_heads, dim, dtype, step=False, rot=None, axes=1, layout="half", per_axis=False,
            norm="rmsnorm", bias=False, packed=False, base=10000.0, far=0):
    return {"name": name, "op": "rotary", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "dtype": dtype, "step": step, "rot": dim if rot is None else rot, "axes": axes, "layout": layout,
            "per_axis": per_axis, "norm": norm, "bias": bias, "packed": packed, "base": base, "far": far}


def listed():
    return [
        # one decoding step of a batch of 8: post norm, residual add, next norm on 8 rows (latency)
        _norms("norms_decode_8x4096_bf16", 8, 1, 4096, "bfloat16"),
        # a long prompt of a wide model whose branches are scaled before the residual add
        _norms("norms_prompt_16384x8192_bf16", 1, 16384, 8192, "bfloat16", branch_scale=0.22),
        # image tokens with per-sample modulation: gate, scale and shift of each of 8 samples, no post norm
        _norms("norms_images_8x1029x1600_fp16", 8, 1029, 1600, "float16", post="none", norm="layernorm", gate="group",
               affine="group", bias=True, offset=1.0),
        # the gated norm of every head behind linear attention: norm(x) * silu(gate), no residual, no second norm
        _norms("norms_head_gate_262144x128_bf16", 1, 262144, 128, "bfloat16", norm="none", gate="element", act="silu",
               residual=False),
        # a training step, norms with weights stored around zero
        _norms("norms_step_16384x4096_bf16", 1, 16384, 4096, "bfloat16", step=True, offset=1.0),
        # a training step on image tokens with per-sample modulation
        _norms("norms_step_images_32x1024x2048_bf16", 32, 1024, 2048, "bfloat16", step=True, post="none", norm="layernorm",
               gate="group", affine="group", bias=True, offset=1.0),
        # a training step in 32 bits, layer norms with biases, a sigmoid gate for every element, an odd row count
        _norms("norms_step_2047x5120_fp32", 1, 2047, 5120, "float32", step=True, post="layernorm", norm="layernorm",
               gate="element", act="sigmoid", bias=True),
        # one decoding step of a batch of 16, far into a long context (latency)
        _rotary("rotary_decode_16x32+8x128_bf16", 16, 32, 8, 128, "bfloat16", packed=True, base=1e6, far=131072),
        # a long prompt of text and image tokens, three axes, heads in place inside the packed projection
        _rotary("rotary_prompt_16384x32+8x128_bf16", 16384, 32, 8, 128, "bfloat16", axes=3, packed=True, base=1e6),
        # video tokens: layer norm with bias on short heads, a frequency ladder for each axis, interleaved pairs
        _rotary("rotary_video_4097x16+16x72_fp16", 4097, 16, 16, 72, "float16", axes=3, layout="interleaved", per_axis=True,
                norm="layernorm", bias=True),
        # a training step of a model with grouped heads, three axes
        _rotary("rotary_step_8192x40+8x128_bf16", 8192, 40, 8, 128, "bfloat16", step=True, axes=3, base=1e6),
        # a training step in 32 bits that rotates the first half of each head
        _rotary("rotary_step_3001x12+4x80_fp32", 3001, 12, 4, 80, "float32", step=True, rot=40),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    step = rng.random() < 0.5
    if rng.random() < 0.55:
        if rng.random() < 0.6:
            hidden = 8 * _log_int(rng, 8, 2048)  # 64 .. 16384
        else:
            hidden = _log_int(rng, 33, 12000)  # any length
        batch = _log_int(rng, 1, 32)
        cap = (1 << 25 if dtype == "float32" else 1 << 26) // (hidden * batch)
        tokens = _log_int(rng, 1, max(1, min(cap, 16384)))
        residual = rng.random() < 0.85
        return _norms("", batch, tokens, hidden, dtype, step,
                      post=rng.choice(["none", "rmsnorm", "rmsnorm", "layernorm"]),
                      norm=rng.choice(["none", "rmsnorm", "rmsnorm", "layernorm"]),
                      gate=rng.choice(["none", "vector", "group", "element"]),
                      act=rng.choice(["none", "sigmoid", "silu", "tanh"]),
                      affine=rng.choice(["none", "vector", "vector", "group"]), bias=rng.random() < 0.4, residual=residual,
                      branch_scale=rng.choice([1.0, 0.22, 0.7071]), residual_scale=rng.choice([1.0, 1.0, 0.9]) if residual else 1.0,
                      offset=rng.choice([0.0, 1.0]))
    dim = rng.choice([32, 64, 72, 80, 96, 112, 128, 128, 192, 256, 50, 90])
    k_heads = _log_int(rng, 1, 16)
    q_heads = k_heads * rng.choice([1, 2, 3, 4, 5, 8])
    cap = (1 << 24 if dtype == "float32" else 1 << 25) // ((q_heads + k_heads) * dim)
    axes = rng.choice([1, 2, 3])
    rot = dim if rng.random() < 0.6 else 2 * rng.randint(max(1, dim // 8), dim // 2)
    return _rotary("", _log_int(rng, 1, max(1, min(cap, 32768))), q_heads, k_heads, dim, dtype, step, rot=rot, axes=axes,
                   layout=rng.choice(["half", "interleaved"]), per_axis=axes > 1 and rng.random() < 0.5,
                   norm=rng.choice(["none", "rmsnorm", "rmsnorm", "layernorm"]), bias=rng.random() < 0.4,
                   packed=rng.random() < 0.5, base=rng.choice([1e4, 5e5, 1e6]), far=rng.choice([0, 0, 4096, 131072]))


# ------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _norms_inputs(c, seed):
    """The tensors of a case by name; absent ones are None."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, b, t, h = _DT[c["dtype"]], c["batch"], c["tokens"], c["hidden"]
    d = {}
    # a few channels of the residual stream are far larger than the rest
    wide = torch.where(torch.rand(h, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    d["x"] = (_randn(g, b, t, h) * 0.8 + 0.05).to(dt)
    d["residual"] = (_randn(g, b, t, h) * wide).to(dt) if c["residual"] else None
    shape = {"none": None, "vector": (h,), "group": (b, h), "element": (b, t, h)}[c["gate"]]
    d["gate"] = None if shape is None else (_randn(g, *shape) * 0.7 + 0.3).to(dt)
    one = 1.0 - c["offset"]
    has_post, has_norm = c["post"] != "none", c["norm"] != "none"
    vec = c["affine"] != "none"
    ashape = (b, h) if c["affine"] == "group" else (h,)
    d["post_weight"] = (one + 0.1 * _randn(g, h)).to(dt) if has_post and vec else None
    d["post_bias"] = (0.1 * _randn(g, h)).to(dt) if has_post and vec and c["bias"] else None
    d["weight"] = (one + 0.1 * _randn(g, *ashape)).to(dt) if has_norm and vec else None
    d["bias"] = (0.1 * _randn(g, *ashape)).to(dt) if has_norm and vec and c["bias"] else None
    if c["step"]:
        d["dy"] = _randn(g, b, t, h).to(dt) if has_norm else None
        d["ds"] = (0.5 * _randn(g, b, t, h)).to(dt)
    return d


_NORMS_LEAVES = ("x", "residual", "gate", "post_weight", "post_bias", "weight", "bias")


def _pairs(c):
    """(axis, inverse frequency) of every rotated pair, as float64 lists: equal sections (the
    first axes take what is left over), one ladder over all pairs or one for each axis."""
    half, axes = c["rot"] // 2, c["axes"]
    sections = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    axis, inv = [], []
    for a, n in enumerate(sections):
        for j in range(n):
            i = j if c["per_axis"] else len(axis)
            inv.append(c["base"] ** (-i / (n if c["per_axis"] else half)))
            axis.append(a)
    return sections, axis, inv


def _positions(c):
    """[axes, tokens]: text tokens with equal positions on all axes, then a grid of patches."""
    n, axes = c["tokens"], c["axes"]
    i = np.arange(n, dtype=np.int64)
    if axes == 1:
        p = i[None] if n > 64 else (i * 977 % 4099)[None]
    else:
        text = n // 4
        j = i - text
        side = max(1, int(math.sqrt(max(1, (n - text) // 4))))
        grid = [text + j // (side * side), text + (j // side) % side, text + j % side]
        p = np.stack([np.where(i < text, i, grid[a]) for a in range(axes)])
    return p + c["far"]


def _rotary_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n, hq, hk, dim = _DT[c["dtype"]], c["tokens"], c["q_heads"], c["k_heads"], c["dim"]
    d = {}
    if c["packed"]:
        qkv = (_randn(g, n, hq + 2 * hk, dim) * 1.3 + 0.1).to(dt)
        d["q"], d["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        d["q"], d["k"] = (_randn(g, n, hq, dim) * 1.3 + 0.1).to(dt), (_randn(g, n, hk, dim) * 1.3 - 0.1).to(dt)
    has = c["norm"] != "none"
    for s in ("q", "k"):
        d[s + "_weight"] = (1.0 + 0.1 * _randn(g, dim)).to(dt) if has else None
        d[s + "_bias"] = (0.1 * _randn(g, dim)).to(dt) if has and c["bias"] else None
    if c["step"]:
        d["dq"], d["dk"] = _randn(g, n, hq, dim).to(dt), _randn(g, n, hk, dim).to(dt)
    d["positions"] = torch.from_numpy(_positions(c)).to("cuda") + seed % 5
    return d


_ROTARY_LEAVES = ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias")


def prepare(case, seed):
    d = _norms_inputs(case, seed) if case["op"] == "norms" else _rotary_inputs(case, seed)
    leaves = _NORMS_LEAVES if case["op"] == "norms" else _ROTARY_LEAVES
    if case["op"] == "rotary":
        sections, axis, inv = _pairs(case)
        if own:
            # the plan a program makes once for its model
            d["rotary"] = _fl().RotaryAxes(case["dim"], sections, base=case["base"], per_axis=case["per_axis"],
                                           layout=case["layout"], device="cuda")
        else:
            d["axis"] = torch.tensor(axis, device="cuda")
            d["inv_freq"] = torch.tensor(inv, dtype=torch.float64, device="cuda")
    if case["step"]:
        for k in leaves:
            if d[k] is not None:
                d[k] = d[k].detach().requires_grad_(True)
    return {"case": case, "t": d, "leaves": [k for k in leaves if d[k] is not None]}


# --------------------------------------------------------------------------------- plain form
def _plain_norm(z, kind, w, b, offset, eps):
    if kind == "none":
        return z
    if kind == "layernorm":
        z = z - z.mean(-1, keepdim=True)
    z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    if w is not None:
        z = z * (offset + w)
    if b is not None:
        z = z + b
    return z


def _plain_act(v, act):
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "tanh":
        return 1.0 - 2.0 / (1.0 + torch.exp(2.0 * v))
    return v


def _f32(t):
    return None if t is None else t.to(torch.float32)


def _rows(t):
    """A per-sample parameter [batch, hidden] next to [batch, tokens, hidden]."""
    return t[:, None, :] if t is not None and t.dim() == 2 else t


def _plain_norms(c, d):
    dt = d["x"].dtype
    n1 = _plain_norm(_f32(d["x"]), c["post"], _f32(d["post_weight"]), _f32(d["post_bias"]), c["offset"], 1e-6)
    s = n1 * c["branch_scale"]
    if d["gate"] is not None:
        s = s * _plain_act(_f32(_rows(d["gate"])), c["act"])
    if d["residual"] is not None:
        s = s + c["residual_scale"] * _f32(d["residual"])
    y = None
    if c["norm"] != "none":
        y = _plain_norm(s, c["norm"], _f32(_rows(d["weight"])), _f32(_rows(d["bias"])), c["offset"], 1e-6).to(dt)
    return y, s.to(dt)


def _plain_rotary(c, d):
    half = c["rot"] // 2
    angle = d["positions"].to(torch.float64)[d["axis"]].t() * d["inv_freq"]  # [tokens, pairs]
    cos, sin = torch.cos(angle).to(torch.float32)[:, None, :], torch.sin(angle).to(torch.float32)[:, None, :]
    out = []
    for s in ("q", "k"):
        z = _plain_norm(_f32(d[s]), c["norm"], _f32(d[s + "_weight"]), _f32(d[s + "_bias"]), 0.0, 1e-6)
        if c["layout"] == "half":
            a, b = z[..., :half], z[..., half:2 * half]
        else:
            a, b = z[..., 0:2 * half:2], z[..., 1:2 * half:2]
        ra, rb = a * cos - b * sin, b * cos + a * sin
        if c["layout"] == "half":
            r = torch.cat([ra, rb], -1)
        else:
            r = torch.stack([ra, rb], -1).reshape(*ra.shape[:-1], 2 * half)
        out.append(torch.cat([r, z[..., 2 * half:]], -1).to(d[s].dtype))
    return tuple(out)


def _own_norms(c, d):
    return _fl().fused_norm_gate_add_norm(
        d["x"], d["residual"], d["gate"], d["post_weight"], d["post_bias"], d["weight"], d["bias"], post_norm=c["post"],
        norm=c["norm"], gate_activation=c["act"], branch_scale=c["branch_scale"], residual_scale=c["residual_scale"],
        weight_offset=c["offset"], post_eps=1e-6, eps=1e-6)


def _own_rotary(c, d):
    return _fl().fused_qk_norm_rotary(d["q"], d["k"], d["positions"], d["rotary"], d["q_weight"], d["k_weight"],
                                      d["q_bias"], d["k_bias"], norm=c["norm"], eps=1e-6)


def run(state):
    c, d = state["case"], state["t"]
    if c["op"] == "norms":
        outs = _own_norms(c, d) if own else _plain_norms(c, d)
        grads = (d.get("dy"), d.get("ds"))
    else:
        outs = _own_rotary(c, d) if own else _plain_rotary(c, d)
        grads = (d.get("dq"), d.get("dk"))
    live = [i for i, o in enumerate(outs) if o is not None]
    res = [outs[i].detach() for i in live]
    if c["step"]:
        res += torch.autograd.grad([outs[i] for i in live], [d[k] for k in state["leaves"]], [grads[i] for i in live])
    return res


# -------------------------------------------------------------------------------------- work
def work(case):
    c = case
    e = 4 if c["dtype"] == "float32" else 2
    if c["op"] == "norms":
        n, h = c["batch"] * c["tokens"] * c["hidden"], c["hidden"]
        second, res, elem = c["norm"] != "none", c["residual"], c["gate"] == "element"
        params = {"none": 0, "vector": h, "group": c["batch"] * h, "element": 0}[c["gate"]]
        if c["affine"] != "none":
            params += (1 + c["bias"]) * ((c["post"] != "none") * h + second * (c["batch"] * h if c["affine"] == "group" else h))
        tensors = 2 + res + elem + second  # x, s, residual, gate, y
        flops = n * (3 * (c["post"] != "none") + 3 * second + 6)
        if c["step"]:
            tensors += 2 + res + elem + second  # ds, dx, d residual, d gate, dy
            params *= 2
            flops *= 3
        return {"bytes": float(e * (n * tensors + params)), "flops": float(flops)}
    n = c["tokens"] * (c["q_heads"] + c["k_heads"]) * c["dim"]
    params = 0 if c["norm"] == "none" else 2 * c["dim"] * (1 + c["bias"])
    k = 2 if c["step"] else 1
    return {"bytes": float(e * (2 * n + params) * k + 8 * c["axes"] * c["tokens"]), "flops": float(n * 9 * (3 if c["step"] else 1))}


# ------------------------------------------------------------------------------- exact values
# From the definitions, in 64 bits, with the gradients written out.
def _x_norm(z, kind, w, b, offset):
    """value, normalized rows, reciprocal deviation, factor"""
    f = torch.ones((), dtype=torch.float64, device=z.device) if w is None else w + offset
    if kind == "none":
        return z, z, None, f
    h = z.shape[-1]
    m = z.sum(-1, keepdim=True) / h if kind == "layernorm" else 0.0
    r = 1.0 / torch.sqrt(((z - m) ** 2).sum(-1, keepdim=True) / h + 1e-6)
    u = (z - m) * r
    return u * f + (0.0 if b is None else b), u, r, f


def _x_norm_grad(dn, u, r, f, kind):
    if kind == "none":
        return dn
    g = dn * f
    g2 = g.mean(-1, keepdim=True) if kind == "layernorm" else 0.0
    return r * (g - g2 - u * (g * u).mean(-1, keepdim=True))


def _x_act(v, act):
    """value and derivative"""
    if act == "none":
        return v, torch.ones_like(v)
    if act == "tanh":
        t = torch.tanh(v)
        return t, 1.0 - t * t
    q = torch.sigmoid(v)
    if act == "sigmoid":
        return q, q * (1.0 - q)
    return v * q, q * (1.0 + v * (1.0 - q))


def _x_like(g, shape):
    """Sum of a full gradient down to a parameter of `shape` ([h], [batch, h] or full)."""
    if len(shape) == 3:
        return g
    return g.sum(1) if len(shape) == 2 else g.sum((0, 1))


def _exact_norms(c, d):
    v = {k: (None if t is None else t.detach().double()) for k, t in d.items()}
    dt = d["x"].dtype
    w2, b2 = _rows(v["weight"]), _rows(v["bias"])
    n1, u1, r1, f1 = _x_norm(v["x"], c["post"], v["post_weight"], v["post_bias"], c["offset"])
    a, da = (1.0, None) if v["gate"] is None else _x_act(_rows(v["gate"]), c["act"])
    s = c["branch_scale"] * a * n1
    if v["residual"] is not None:
        s = s + c["residual_scale"] * v["residual"]
    y, u2, r2, f2 = _x_norm(s, c["norm"], w2, b2, c["offset"])
    out = ([] if c["norm"] == "none" else [y]) + [s]
    if c["step"]:
        ds = v["ds"]
        if c["norm"] != "none":
            ds = ds + _x_norm_grad(v["dy"], u2, r2, f2, c["norm"])
        e = ds * c["branch_scale"]
        out.append(_x_norm_grad(e * a, u1, r1, f1, c["post"]))
        if v["residual"] is not None:
            out.append(ds * c["residual_scale"])
        if v["gate"] is not None:
            out.append(_x_like(e * n1 * da, d["gate"].shape))
        for k, g in (("post_weight", lambda: e * a * u1), ("post_bias", lambda: e * a + 0.0 * u1),
                     ("weight", lambda: v["dy"] * u2), ("bias", lambda: v["dy"])):
            if v[k] is not None:
                out.append(_x_like(g(), d[k].shape))
    return out


def _exact_rotary(c, d):
    _, axis, inv = _pairs(c)
    half = c["rot"] // 2
    ang = np.stack([d["positions"][a].cpu().numpy().astype(np.float64) * f for a, f in zip(axis, inv)], 1)
    rot = torch.from_numpy(np.exp(1j * ang)).to("cuda")[:, None, :]
    lo = torch.arange(half, device="cuda") * (1 if c["layout"] == "half" else 2)
    hi = lo + (half if c["layout"] == "half" else 1)

    def turn(z, by):
        w = torch.complex(z[..., lo], z[..., hi]) * by
        o = z.clone()
        o[..., lo], o[..., hi] = w.real, w.imag
        return o

    outs, grads = [], {}
    for s in ("q", "k"):
        w, b = (None if d[s + p] is None else d[s + p].detach().double() for p in ("_weight", "_bias"))
        n, u, r, f = _x_norm(d[s].detach().double(), c["norm"], w, b, 0.0)
        outs.append(turn(n, rot))
        if c["step"]:
            dn = turn(d["d" + s].double(), rot.conj())
            grads[s] = _x_norm_grad(dn, u, r, f, c["norm"])
            grads[s + "_weight"], grads[s + "_bias"] = (dn * u).sum((0, 1)), dn.sum((0, 1))
    return outs + ([grads[k] for k in _ROTARY_LEAVES if d[k] is not None] if c["step"] else [])


def exact(case, seed):
    with torch.no_grad():
        if case["op"] == "norms":
            return _exact_norms(case, _norms_inputs(case, seed))
        return _exact_rotary(case, _rotary_inputs(case, seed))
