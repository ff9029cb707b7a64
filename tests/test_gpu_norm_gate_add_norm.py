"""fused_norm_gate_add_norm (norm -> gate -> scaled residual add -> norm) against the formula in
64 bits: values, all seven gradients, differences, strides, streams, graphs, refusals.  The
bounds are those of block_norms_ref."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import block_norms_ref as R

if torch.cuda.is_available():
    import fused_layernorm as fl

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(shape, dtype, post="rmsnorm", norm="rmsnorm", gate="none", act="none", affine="vector", bias=False, residual=True,
         off=0.0, seed=0, ba=1.0, ra=1.0):
    g = torch.Generator().manual_seed(seed)
    h = shape[-1]
    rn = lambda *s: torch.randn(*s, generator=g)
    one = 1.0 - off
    grouped = (shape[0], h)
    t = dict.fromkeys(R.NAMES)
    t["input"] = rn(*shape) * 0.9 + 0.2
    if residual:
        t["residual"] = rn(*shape) * 1.5
    if gate != "none":
        t["gate"] = 0.3 + 0.8 * rn(*{"vector": (h,), "group": grouped, "element": shape}[gate])
    if post != "none" and affine != "none":
        t["post_weight"] = one + 0.2 * rn(h)
        t["post_bias"] = 0.2 * rn(h) if bias else None
    if norm != "none" and affine != "none":
        t["weight"] = one + 0.2 * rn(*(grouped if affine == "group" else (h,)))
        t["bias"] = 0.2 * rn(*(grouped if affine == "group" else (h,))) if bias else None
    t = {k: None if v is None else v.to(dtype).cuda() for k, v in t.items()}
    dy, ds = (rn(*shape).to(dtype).cuda() for _ in range(2))
    conf = dict(post_norm=post, norm=norm, gate_activation=act, branch_scale=ba, residual_scale=ra, weight_offset=off)
    return t, (dy if norm != "none" else None), ds, conf


def call(t, conf):
    return fl.fused_norm_gate_add_norm(*[t[n] for n in R.NAMES], **conf, post_eps=R.EPS1, eps=R.EPS2)


def bounds(t, dy, ds, conf):
    d = lambda v: None if v is None else v.detach().double()
    return R.nga_bounds({k: d(v) for k, v in t.items()}, d(dy), d(ds), t["input"].dtype, conf["post_norm"], conf["norm"],
                        conf["gate_activation"], conf["branch_scale"], conf["residual_scale"], conf["weight_offset"])


def check_case(t, dy, ds, conf):
    """Values without and with autograd, and all gradients."""
    want = bounds(t, dy, ds, conf)
    y, s = call(t, conf)
    assert (y is None) == (conf["norm"] == "none")
    R.check(s, want["sum"], "sum")
    if y is not None:
        R.check(y, want["y"], "y")
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    y2, s2 = call({k: leaves.get(k) for k in t}, conf)
    assert torch.equal(s, s2) and (y is None or torch.equal(y, y2))
    outs, grads = ([s2], [ds]) if y is None else ([y2, s2], [dy, ds])
    got = torch.autograd.grad(outs, list(leaves.values()), grads, retain_graph=True)
    for k, g in zip(leaves, got):
        assert g.dtype == t[k].dtype
        R.check(g, want["grads"][k], "d" + k)
    again = torch.autograd.grad(outs, list(leaves.values()), grads)
    for a, b in zip(got, again):
        assert torch.equal(a, b)  # sums in a fixed order


SHAPES = [((1, 1), F32), ((3, 7), BF16), ((2, 5, 33), F16), ((1, 64), BF16), ((5, 128), F32), ((4, 9, 128), BF16),
          ((300, 128), F16), ((17, 1000), BF16), ((2, 33, 768), F16), ((129, 1024), BF16), ((3, 41, 1600), BF16),
          ((2, 70, 2048), BF16), ((7, 4096), F32), ((150, 4096), BF16), ((2, 3, 5, 1152), F32), ((33, 5120), F16),
          ((65, 8192), BF16), ((9, 8192), F32), ((5, 12289), BF16), ((3, 16384), F16), ((4, 20000), F32)]
KINDS = [dict(post="rmsnorm", norm="rmsnorm"), dict(post="layernorm", norm="layernorm", bias=True),
         dict(post="none", norm="rmsnorm"), dict(post="rmsnorm", norm="none"), dict(post="none", norm="layernorm", bias=True),
         dict(post="layernorm", norm="rmsnorm", bias=True)]
GATES = [dict(gate="none"), dict(gate="vector", act="tanh"), dict(gate="group"), dict(gate="element", act="silu"),
         dict(gate="element", act="sigmoid"), dict(gate="group", act="sigmoid", affine="group")]


@pytest.mark.parametrize("shape,dtype", SHAPES, ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("i", range(6))
def test_values_and_gradients(shape, dtype, i):
    """Every shape with six pairs of norm kinds and gate kinds, shifted from shape to shape so
    that all pairs meet."""
    j = SHAPES.index((shape, dtype))
    kind, gate = KINDS[i], GATES[(i + j) % 6]
    check_case(*make(shape, dtype, **kind, **gate, off=float((i + j) % 2), seed=100 * j + i, ba=0.7 if i % 2 else 1.0,
                     ra=0.9 if i % 3 == 0 else 1.0, residual=(i + j) % 5 != 0))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("affine", ["none", "vector", "group"])
@pytest.mark.parametrize("gate", ["none", "vector", "group", "element"])
def test_groups_of_every_length(dtype, affine, gate):
    """Per-sample vectors with samples of one row, of a few, and longer than a slot."""
    for i, (b, n, h) in enumerate([(6, 1, 256), (5, 3, 520), (3, 131, 96), (2, 700, 64)]):
        check_case(*make((b, n, h), dtype, post="rmsnorm", norm="layernorm", bias=True, gate=gate, affine=affine,
                         act="tanh" if gate != "none" else "none", off=1.0, seed=i))


@pytest.mark.parametrize("shape,dtype", [((3, 8200), F32), ((2, 11, 9984), F16), ((200, 10007), BF16), ((2, 90, 16384), BF16),
                                         ((5, 16383), F32), ((3, 16392), F16)], ids=lambda v: str(v).replace("torch.", ""))
def test_long_rows(shape, dtype):
    """Rows that two CTAs share in the backward, and rows beyond those; whole vectors and not."""
    for i in range(6):
        check_case(*make(shape, dtype, **KINDS[i], **GATES[(i + len(shape)) % 6], off=float(i % 2), seed=i, ba=0.7))


@pytest.mark.parametrize("shape,dtype", [((2, 39, 5120), BF16), ((2, 39, 5120), F32), ((5, 31, 2560), F32), ((5, 31, 2560), F16),
                                         ((301, 5120), F32), ((3, 100, 1280), BF16)], ids=lambda v: str(v).replace("torch.", ""))
def test_whole_rows_of_five_times_a_power_of_two(shape, dtype):
    """Every pair of norm kinds and every kind of gate, with a residual and with both gradients."""
    for i in range(6):
        for j in range(6):
            check_case(*make(shape, dtype, **KINDS[i], **GATES[j], off=float(i % 2), seed=6 * i + j, ba=0.7))


@pytest.mark.parametrize("h", [1, 2, 3, 5, 9, 31, 65, 130, 257, 333, 511, 1001, 2050, 2777, 4100, 5121, 6007, 7998])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_start_anywhere_in_a_vector(h, dtype):
    """Row lengths that are not whole vectors: every class of starting places, groups shorter than
    the number of classes, neighbours with infinities in the same vectors."""
    i = h % 6
    for b, n in ((1, 67), (5, 3), (9, 1)):
        check_case(*make((b, n, h), dtype, **KINDS[i], **GATES[(i + n) % 6], off=float(h % 2), seed=h + n))
    t, dy, ds, conf = make((33, h), dtype, post="layernorm", norm="layernorm", bias=True)
    want = call(t, conf)
    grads = lambda v: torch.autograd.grad(call(v, conf), [v["input"], v["residual"]], [dy, ds])
    leaves = lambda v: {k: (None if x is None else x.detach().requires_grad_(True)) for k, x in v.items()}
    g = grads(leaves(t))
    bad = {k: (None if v is None else v.clone()) for k, v in t.items()}
    bad["input"][1::2] = float("inf")
    bad["residual"][1::2] = float("nan")
    got, gb = call(bad, conf), grads(leaves(bad))
    for a, b in zip((*got, *gb), (*want, *g)):
        assert torch.equal(a[::2], b[::2])


def test_more_groups_than_partial_rows_and_many_rows():
    check_case(*make((1500, 2, 72), BF16, gate="group", affine="group", seed=3))
    check_case(*make((70001, 16), F32, bias=True, post="layernorm", norm="layernorm", seed=4))
    check_case(*make((40000, 128), BF16, gate="element", act="silu", norm="none", residual=False, seed=5))


def test_only_some_gradients():
    t, dy, ds, conf = make((37, 640), BF16, gate="vector", act="silu", bias=True, post="layernorm", norm="layernorm")
    want = bounds(t, dy, ds, conf)["grads"]
    for names in (["input"], ["residual"], ["weight"], ["post_bias"], ["gate"], ["bias", "input"], ["post_weight", "residual"]):
        s = {k: (v.detach().requires_grad_(k in names) if v is not None else None) for k, v in t.items()}
        y, su = call(s, conf)
        outs = [o for o in (y, su) if o.requires_grad]
        got = torch.autograd.grad([y, su], [s[n] for n in names], [dy, ds])
        assert len(outs) == 2
        for n, g in zip(names, got):
            R.check(g, want[n], n)


def test_gradient_of_one_output_alone():
    t, dy, ds, conf = make((21, 768), F32, gate="group", act="none")
    for use in ("y", "sum"):
        s = {k: (v.detach().requires_grad_(True) if v is not None else None) for k, v in t.items()}
        y, su = call(s, conf)
        (y if use == "y" else su).backward(dy if use == "y" else ds)
        want = bounds(t, dy if use == "y" else None, ds if use == "sum" else None, conf)["grads"]
        for k, v in s.items():
            if v is None:
                continue
            if use == "sum" and k == "weight":
                assert v.grad is None or not bool(v.grad.any())
            else:
                R.check(v.grad, want[k], k)


def test_gradients_against_differences():
    """(L(+h d) - L(-h d)) / 2h of the kernel's own outputs, L = <dy, y> + <ds, sum> in 64 bits,
    against <gradient, d>.  The difference may be off by the outputs' rounding over h, and by the
    truncation that the same difference of the 64-bit formula shows."""
    for kw in (dict(gate="vector", act="tanh", post="layernorm", norm="layernorm", bias=True),
               dict(gate="element", act="silu"), dict(gate="group", act="sigmoid", affine="group", off=1.0)):
        t, dy, ds, conf = make((3, 5, 192), F32, seed=11, ra=0.9, ba=0.8, **kw)
        leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
        y, s = call({k: leaves.get(k) for k in t}, conf)
        grads = dict(zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [dy, ds])))
        formula = {k: v.detach().double().requires_grad_(True) for k, v in leaves.items()}

        def exact(v):
            yy, ss = R.nga_formula(*[v.get(n) for n in R.NAMES], conf["post_norm"], conf["norm"], conf["gate_activation"],
                                   conf["branch_scale"], conf["residual_scale"], conf["weight_offset"])
            return (dy.double() * yy).sum() + (ds.double() * ss).sum()

        slope = dict(zip(formula, torch.autograd.grad(exact(formula), list(formula.values()))))
        h = 2.0 ** -7
        g = torch.Generator().manual_seed(5)
        for k in leaves:
            d = torch.randn(leaves[k].shape, generator=g).cuda()
            vals, exacts = [], []
            for sign in (1, -1):
                moved = {n: (v.detach() + sign * h * d if n == k else v.detach()) for n, v in leaves.items()}
                yy, ss = call({n: moved.get(n) for n in t}, conf)
                vals.append((dy.double() * yy.double()).sum() + (ds.double() * ss.double()).sum())
                exacts.append(exact({n: v.double() for n, v in moved.items()}))
            got, trunc = (vals[0] - vals[1]) / (2 * h), (exacts[0] - exacts[1]) / (2 * h) - (slope[k] * d.double()).sum()
            noise = 2.0 ** -24 * 60 * ((dy * y).double().abs().sum() + (ds * s).double().abs().sum()) / h
            assert (got - (grads[k].double() * d.double()).sum()).abs() <= noise + 1.01 * trunc.abs(), k


def test_strides_and_offsets():
    """Views: transposed input, a slice of a wider tensor, parameters with a step, unaligned
    storage offsets, gradients that arrive expanded or transposed."""
    t, dy, ds, conf = make((6, 40, 264), BF16, gate="element", act="silu", seed=7)
    want = bounds(t, dy, ds, conf)
    v = dict(t)
    v["input"] = t["input"].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(6, 40, 300, dtype=BF16, device="cuda")
    wide[..., 3:267] = t["residual"]
    v["residual"] = wide[..., 3:267]
    flat = torch.zeros(6 * 40 * 264 + 1, dtype=BF16, device="cuda")
    flat[1:] = t["gate"].reshape(-1)
    v["gate"] = flat[1:].view(6, 40, 264)  # 2 bytes off any vector boundary
    two = torch.zeros(264, 2, dtype=BF16, device="cuda")
    two[:, 0] = t["weight"]
    v["weight"] = two[:, 0]
    v = {k: (None if x is None else x.detach().requires_grad_(True)) for k, x in v.items()}
    y, s = call(v, conf)
    R.check(y, want["y"], "y")
    R.check(s, want["sum"], "sum")
    got = torch.autograd.grad([y, s], [v[k] for k in t if t[k] is not None],
                              [dy.transpose(0, 1).contiguous().transpose(0, 1), ds])
    for k, g in zip([k for k in t if t[k] is not None], got):
        R.check(g, want["grads"][k], k)
    # a gradient that is one value seen everywhere
    one = torch.ones((), dtype=BF16, device="cuda").expand(6, 40, 264)
    y, s = call(v, conf)
    g = torch.autograd.grad(y, v["residual"], one)[0]
    R.check(g, bounds(t, one, None, conf)["grads"]["residual"], "dresidual")


def test_shapes_of_gate_and_modulation():
    """[batch, 1, hidden] and [1, hidden] forms, a batch of one, rows without a batch."""
    for gshape in ((4, 96), (4, 1, 96), (1, 96), (1, 1, 96), (96,)):
        t, dy, ds, conf = make((4, 6, 96), F32)
        t["gate"] = torch.randn(*gshape, device="cuda")
        ref = dict(t)
        ref["gate"] = t["gate"].reshape(gshape[0], 96) if gshape[0] == 4 else t["gate"].reshape(96)
        want = bounds(ref, dy, ds, conf)
        gate = t["gate"].requires_grad_(True)
        y, s = call(t, conf)
        R.check(y, want["y"], "y")
        g = torch.autograd.grad([y, s], gate, [dy, ds])[0]
        assert g.shape == gate.shape
        v, tol = want["grads"]["gate"]
        R.check(g.reshape(v.shape), (v, tol), "dgate")
    t, dy, ds, conf = make((96,), F32)
    check_case(t, dy, ds, conf)


def test_empty():
    for shape in ((0, 64), (3, 0, 64), (0, 5, 64)):
        t, dy, ds, conf = make(shape, BF16, gate="vector", bias=True, post="layernorm", norm="layernorm")
        v = {k: (None if x is None else x.detach().requires_grad_(True)) for k, x in t.items()}
        y, s = call(v, conf)
        assert y.shape == shape and s.shape == shape
        (y.sum() + s.sum()).backward()
        for k in ("gate", "post_weight", "post_bias", "weight", "bias"):
            assert v[k].grad.shape == (64,) and not bool(v[k].grad.any())
    t, dy, ds, conf = make((4, 0, 64), F32, gate="group", affine="group", bias=True)
    v = {k: (None if x is None else x.detach().requires_grad_(True)) for k, x in t.items()}
    y, s = call(v, conf)
    (y.sum() + s.sum()).backward()
    for k in ("gate", "weight", "bias"):
        assert v[k].grad.shape == (4, 64) and not bool(v[k].grad.any())


def test_rows_of_zeros_of_one_value_and_of_infinities():
    """Rows of zeros and constant rows have values and gradients of the formula; a row with an
    infinity or NaN spoils that row only."""
    t, dy, ds, conf = make((6, 256), F32, post="layernorm", norm="layernorm", bias=True)
    t["input"][1] = 0
    t["input"][2] = 3.0
    check_case(t, dy, ds, conf)
    clean = call(t, conf)
    bad = dict(t)
    bad["input"] = t["input"].clone()
    bad["input"][3, 5] = float("inf")
    bad["input"][4, 7] = float("nan")
    y, s = call(bad, conf)
    keep = [0, 1, 2, 5]
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(s[keep], clean[1][keep])
    assert not bool(torch.isfinite(y[[3, 4]]).all(-1).any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gates_far_out(dtype):
    """Saturated gates: activations at +-80 and +-1000 are 0 or 1 (silu: 0 or the gate), and no NaN."""
    t, dy, ds, conf = make((4, 128), dtype, norm="none", gate="element", act="sigmoid", residual=False)
    t["gate"][:] = torch.tensor([-1000.0, -80.0, 80.0, 1000.0])[:, None].to(dtype)
    for act in ("sigmoid", "silu", "tanh"):
        conf["gate_activation"] = act
        check_case(t, dy, ds, conf)


def test_streams_and_devices():
    t, dy, ds, conf = make((300, 1024), BF16, gate="vector")
    want = call(t, conf)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        st.wait_stream(torch.cuda.default_stream())
        got = call(t, conf)
    torch.cuda.default_stream().wait_stream(st)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_graphs_replayed_in_turn():
    """Forward and backward captured into two graphs with their own inputs, replayed by turns and
    after the inputs change."""
    conf = None
    graphs = []
    for seed in (1, 2):
        t, dy, ds, conf = make((4, 200, 512), BF16, gate="group", affine="group", bias=True, post="layernorm",
                               norm="layernorm", seed=seed)
        leaves = {k: v.detach().clone().requires_grad_(True) for k, v in t.items() if v is not None}

        def step(leaves=leaves, dy=dy, ds=ds):
            y, s = call({k: leaves.get(k) for k in R.NAMES}, conf)
            return (y, s) + torch.autograd.grad([y, s], list(leaves.values()), [dy, ds])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, leaves, out, step))
    for turn in range(3):
        for g, leaves, out, step in graphs:
            with torch.no_grad():
                leaves["input"].mul_(0.9).add_(0.05)
            g.replay()
        torch.cuda.synchronize()
        for g, leaves, out, step in graphs:
            for a, b in zip(out, step()):
                assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """More than 2**31 elements in each tensor: the last rows and the sums over all rows."""
    rows, h = 262200, 8200  # 2.15e9 elements
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, h, dtype=BF16, device="cuda").normal_(generator=g)
    r = torch.empty(rows, h, dtype=BF16, device="cuda").normal_(generator=g)
    w1, w2 = (torch.randn(h, device="cuda", generator=g).to(BF16) for _ in range(2))
    leaves = [v.requires_grad_(True) for v in (x, r, w1, w2)]
    y, s = fl.fused_norm_gate_add_norm(x, r, None, w1, None, w2, post_eps=R.EPS1, eps=R.EPS2)
    one = torch.ones((), dtype=BF16, device="cuda").expand_as(y)
    dx, dr, dw1, dw2 = torch.autograd.grad([y], leaves, [one])
    for part in (slice(0, 2), slice(rows // 2, rows // 2 + 2), slice(rows - 2, rows)):
        t = dict.fromkeys(R.NAMES)
        t.update(input=x[part], residual=r[part], post_weight=w1, weight=w2)
        conf = dict(post_norm="rmsnorm", norm="rmsnorm", gate_activation="none", branch_scale=1.0, residual_scale=1.0, weight_offset=0.0)
        want = bounds(t, one[part], None, conf)
        R.check(y[part], want["y"], "y"), R.check(s[part], want["sum"], "sum")
        R.check(dx[part], want["grads"]["input"], "dx"), R.check(dr[part], want["grads"]["residual"], "dresidual")
    # dweight = sum of sh: |sh| sums to about 0.8 rows, each term is good to 2**-14 (e24 of the bounds
    # at this row length), the sum's rounding is half a step of bf16
    total = torch.zeros(h, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    with torch.no_grad():
        for i in range(0, rows, 8740):
            v = R.norm_of(x[i:i + 8740].double(), "rmsnorm", w1.double(), None, 0.0, R.EPS1)[0] + r[i:i + 8740].double()
            sh = v / torch.sqrt((v * v).mean(-1, keepdim=True) + R.EPS2)
            total += sh.sum(0)
            size += sh.abs().sum(0)
    R.check(dw2, (total, R.u_of(BF16) * total.abs() + (2.0 ** -14 + (64 + rows / 64) * 2.0 ** -24) * size), "dweight")


def test_refusals():
    t, dy, ds, conf = make((4, 6, 96), BF16, gate="vector")
    ok = lambda **kw: call({**t, **{k: v for k, v in kw.items() if k in t}}, {**conf, **{k: v for k, v in kw.items() if k not in t}})
    ok()
    bad = [dict(residual=t["residual"][:, :5]), dict(residual=t["residual"].float()), dict(gate=t["gate"][:95]),
           dict(gate=torch.zeros(6, 96, dtype=BF16, device="cuda")), dict(gate=torch.zeros(4, 2, 96, dtype=BF16, device="cuda")),
           dict(weight=torch.zeros(4, 6, 96, dtype=BF16, device="cuda")), dict(weight=t["weight"].cpu()),
           dict(post_weight=torch.zeros(4, 96, dtype=BF16, device="cuda")),
           dict(bias=torch.zeros(4, 96, dtype=BF16, device="cuda")),  # next to a weight of [hidden]
           dict(post_norm="none"), dict(norm="none"),
           dict(input=t["input"].cpu())]
    for kw in bad:
        with pytest.raises(RuntimeError):
            ok(**kw)
    with pytest.raises(NotImplementedError):
        fl.fused_norm_gate_add_norm(torch.zeros(2, 8, dtype=torch.float64, device="cuda"))
    for kw in (dict(post_norm="batch"), dict(norm=3), dict(gate_activation="relu")):
        with pytest.raises(ValueError):
            ok(**kw)
    x = t["input"].detach().requires_grad_(True)
    y, s = fl.fused_norm_gate_add_norm(x)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_tensors_changed_before_the_backward():
    """The backward reads the inputs, so changing one is refused; the outputs belong to the caller."""
    t, dy, ds, conf = make((4, 96), F32)
    want = bounds(t, dy, ds, conf)["grads"]
    x, r = (t[n].detach().clone().requires_grad_(True) for n in ("input", "residual"))
    y, s = call({**t, "input": x, "residual": r}, conf)
    with torch.no_grad():
        y.zero_(), s.zero_()
    got = torch.autograd.grad([y, s], [x, r], [dy, ds], retain_graph=True)
    R.check(got[0], want["input"], "dx"), R.check(got[1], want["residual"], "dresidual")
    with torch.no_grad():
        r.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad([y, s], [x, r], [dy, ds])


def test_module_and_compile():
    torch.manual_seed(0)
    m = fl.FusedNormGateAddNorm(320, layer_scale=0.5, weight_offset=1.0, device="cuda", dtype=BF16)
    assert set(m.state_dict()) == {"post_weight", "weight", "gate"} and not bool(m.weight.any())
    x, r = (torch.randn(3, 11, 320, device="cuda", dtype=BF16) for _ in range(2))
    y, s = m(x, r)
    y2, s2 = fl.fused_norm_gate_add_norm(x, r, m.gate, m.post_weight, None, m.weight, None, weight_offset=1.0)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    fn = torch.compile(lambda *a: m(*a), fullgraph=True, backend="aot_eager")
    xa, xb = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    (m(xa, r)[0].float().sum()).backward()
    eager = [p.grad.clone() for p in m.parameters()]
    for p in m.parameters():
        p.grad = None
    y3, s3 = fn(xb, r)
    assert torch.equal(y3, y) and torch.equal(s3, s)
    y3.float().sum().backward()
    assert torch.equal(xa.grad, xb.grad)
    for p, g in zip(m.parameters(), eager):
        assert torch.equal(p.grad, g)
