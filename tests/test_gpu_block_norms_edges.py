"""Edges of the block norms: infinities where a formula keeps them to themselves, angles next to
quarter turns, work queued on another stream."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import block_norms_ref as R

if torch.cuda.is_available():
    import fused_layernorm as fl

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("shape", [(1, 3, 64), (2, 5, 128), (3, 67, 96), (4, 1, 128), (2, 9, 33), (1, 201, 256)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("gate", ["vector", "group"])
def test_infinite_inputs_in_the_gradient_of_a_shared_gate(shape, dtype, gate):
    """dgate = act'(gate) * sum of branch_scale * dsum * x without a norm in front: an infinity in the
    last row of a sample makes an infinity of its column, not NaN, and touches no other column.  The
    rows do not fill the row groups of a block."""
    b, n, h = shape
    g = torch.Generator().manual_seed(h + n)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    x, r, ds, gt = rn(*shape), rn(*shape), rn(*shape), rn(*((h,) if gate == "vector" else (b, h)))
    x[-1, -1, 3], x[0, -1, h - 1] = float("inf"), float("-inf")
    ds[-1, -1, 3], ds[0, -1, h - 1] = 0.5, 1.5
    leaf = gt.clone().requires_grad_(True)
    _, s = fl.fused_norm_gate_add_norm(x, r, leaf, post_norm=None, norm=None, gate_activation="sigmoid", branch_scale=0.7)
    got = torch.autograd.grad(s, leaf, ds)[0]
    t = dict.fromkeys(R.NAMES)
    t.update(input=x.double(), residual=r.double(), gate=gt.double())
    want, tol = R.nga_bounds(t, None, ds.double(), dtype, "none", "none", "sigmoid", 0.7, 1.0, 0.0)["grads"]["gate"]
    fin = torch.isfinite(want)
    assert int((~fin).sum()) == 2 and bool((want[~fin].abs() == math.inf).all())
    assert torch.equal(got[~fin].double(), want[~fin])
    R.check(got[fin], (want[fin], tol.expand(want.shape)[fin]), "dgate")


@pytest.mark.parametrize("dim,pairs", [(128, 32), (80, 20), (72, 16), (50, 10), (51, 20), (64, 0), (256, 64), (510, 100)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_infinities_behind_the_rotated_part(dim, pairs, dtype, layout):
    """Elements behind the rotated part pass without a norm as they are, in both directions: an
    infinity or NaN among them stays where it is.  With a norm the row's other elements are zero
    (rstd is 0), not NaN."""
    rot = fl.RotaryAxes(dim, pairs, layout=layout, magnitude=1.25)
    pos = torch.arange(9, device="cuda") * 37
    g = torch.Generator().manual_seed(dim)
    q, dq = (torch.randn(9, 3, dim, generator=g).to(dtype).cuda() for _ in range(2))
    odd = {2 * pairs: float("inf"), dim - 1: float("nan"), 2 * pairs + (dim - 2 * pairs) // 2: float("-inf")}

    def spoil(v):
        v = v.clone()
        for c, w in odd.items():
            v[c % 9, 1, c] = w
        return v

    def run(q, dq):
        leaf = q.clone().requires_grad_(True)
        o, _ = fl.fused_qk_norm_rotary(leaf, None, pos, rot, norm=None)
        return o.detach(), torch.autograd.grad(o, leaf, dq)[0]

    for got, clean in zip(run(spoil(q), spoil(dq)), run(q, dq)):
        assert torch.equal(torch.nan_to_num(got, nan=77.0), torch.nan_to_num(spoil(clean), nan=77.0))
    one = q.clone()
    one[4, 2, dim - 1] = float("inf")
    o, _ = fl.fused_qk_norm_rotary(one, None, pos, rot)
    assert bool(torch.isnan(o[4, 2, dim - 1])) and not bool(o[4, 2, :dim - 1].any())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_cosines_and_sines_keep_their_own_bits(layout):
    """Every cosine and sine is good relative to itself, next to its zeros too.  The fraction of a turn
    is an exact integer; what is left of it behind whole quarter turns is rounded to 24 bits, which
    moves a sine or cosine by 2**-24 of itself at most (x cot x <= 1 and x tan x <= pi / 4 up to an
    eighth of a turn), and sine and cosine are good to one unit in the last place, 2**-23."""
    freq = [math.pi / 2, math.pi, math.pi / 4, 3 * math.pi / 2, 2 * math.pi / 3, 1.0, 1e-3, math.pi * (1 + 2.0 ** -30)]
    n = len(freq)
    rot = fl.RotaryAxes(2 * n, n, inv_freq=freq, layout=layout)
    g = torch.Generator().manual_seed(0)
    pos = torch.cat([torch.arange(-20, 20), torch.randint(-2 ** 40, 2 ** 40, (3000,), generator=g)]).cuda()
    lo, hi = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, None, 2), slice(1, None, 2))
    q = torch.zeros(len(pos), 1, 2 * n, device="cuda")
    q[..., lo] = 1.0  # rotates to (cos, sin)
    out = fl.fused_qk_norm_rotary(q, None, pos, rot, norm=None)[0][:, 0].cpu().double()
    turns = [int(v) % 2 ** 64 for v in rot.turns.tolist()]
    quarter, rest = [], []
    for p in pos.tolist():
        for t in turns:
            f = p * t % 2 ** 64
            quarter.append((f + 2 ** 61 >> 62) % 4)
            rest.append(((f + 2 ** 61) % 2 ** 62 - 2 ** 61) / 2 ** 64)
    k, a = torch.tensor(quarter).view(-1, n), torch.tensor(rest, dtype=torch.float64).view(-1, n) * (2 * math.pi)
    c, s = torch.cos(a), torch.sin(a)
    cos = torch.stack([c, -s, -c, s]).gather(0, k[None])[0]
    sin = torch.stack([s, c, -s, -c]).gather(0, k[None])[0]
    for got, want in ((out[:, lo], cos), (out[:, hi], sin)):
        assert ((got - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all(), ((got - want).abs() / want.abs()).max() * 2 ** 24


def behind(stream, fn, *bufs):
    """Runs fn on `stream` behind a kernel that takes some 20 ms and a copy of the real inputs into
    buffers of zeros: what is launched anywhere else finds the zeros."""
    live = [torch.zeros_like(b) for b in bufs]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(40_000_000)
        for a, b in zip(live, bufs):
            a.copy_(b)
        out = fn(*live)
    stream.synchronize()
    return out


def test_norm_gate_add_norm_follows_the_current_stream():
    g = torch.Generator().manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    w1, w2, gate = rn(1024), rn(1024), rn(1024)

    def step(x, r, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w1, w2, gate)]
        y, s = fl.fused_norm_gate_add_norm(leaves[0], leaves[1], leaves[4], leaves[2], None, leaves[3])
        return (y, s, *torch.autograd.grad(y, leaves, dy))

    bufs = [rn(300, 1024) for _ in range(3)]
    want = step(*bufs)
    for a, b in zip(behind(torch.cuda.Stream(), step, *bufs), want):
        assert torch.equal(a, b)


def test_qk_norm_rotary_follows_the_current_stream():
    g = torch.Generator().manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    w = rn(128)
    rot = fl.RotaryAxes(128, (16, 24, 24))
    pos = torch.arange(3 * 200, device="cuda").view(3, 200)

    def step(q, k, dq, pos):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, w)]
        o = fl.fused_qk_norm_rotary(leaves[0], leaves[1], pos, rot, leaves[2], leaves[2])
        grads = torch.autograd.grad(o[0], leaves[::2], dq)
        with torch.no_grad():
            place = fl.fused_qk_norm_rotary_(q, k, pos, rot, w, w)
        return (*o, *grads, *place)

    bufs = [rn(200, 8, 128), rn(200, 2, 128), rn(200, 8, 128), pos]
    want = step(*[b.clone() for b in bufs])
    for a, b in zip(behind(torch.cuda.Stream(), step, *bufs), want):
        assert torch.equal(a, b)


def test_in_place_rotary_inside_a_compiled_function():
    """The in-place form breaks the graph of torch.compile and runs between its parts."""
    rot, pos = fl.RotaryAxes(64, 32), torch.arange(7, device="cuda")
    qkv = torch.randn(7, 6, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(0))

    def fn(qkv):
        qkv = qkv * 2.0
        q, k = fl.fused_qk_norm_rotary_(qkv[:, :4], qkv[:, 4:5], pos, rot)
        return q + 1.0, k, qkv

    with torch.no_grad():
        for a, b in zip(torch.compile(fn, backend="aot_eager")(qkv), fn(qkv)):
            assert torch.equal(a, b)


def test_backward_while_another_thread_changes_the_sm_reserve():
    """A backward plans with the settings of one moment: beside a thread that moves the reserve it is
    right, or refused for the workspace that was asked for at another moment."""
    import threading
    from fused_layernorm import _capi as capi
    g = torch.Generator().manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    t = dict.fromkeys(R.NAMES)
    t.update(input=rn(900, 512), residual=rn(900, 512), post_weight=rn(512), weight=rn(512))
    dy = rn(900, 512)
    leaves = {k: v.requires_grad_(True) for k, v in t.items() if v is not None}
    want = R.nga_bounds({k: None if v is None else v.detach().double() for k, v in t.items()}, dy.double(), None, BF16, "rmsnorm",
                        "rmsnorm", "none", 1.0, 1.0, 0.0)["grads"]
    lib, stop = capi.lib(), threading.Event()

    def move():
        while not stop.is_set():
            for n in (0, 100, 40, 140):
                lib.fln_set_sm_reserve(n)

    mover, right = threading.Thread(target=move), 0
    mover.start()
    try:
        for _ in range(200):
            y, s = fl.fused_norm_gate_add_norm(t["input"], t["residual"], None, t["post_weight"], None, t["weight"], None,
                                               post_eps=R.EPS1, eps=R.EPS2)
            try:
                got = torch.autograd.grad(y, list(leaves.values()), dy)
            except RuntimeError as e:
                assert "workspace" in str(e)
                continue
            right += 1
            for k, v in zip(leaves, got):
                R.check(v, want[k], k)
    finally:
        stop.set(), mover.join()
        lib.fln_set_sm_reserve(0)
    assert right > 0


@pytest.mark.parametrize("post", [None, "layernorm"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_unaligned_bias_beside_aligned_tensors(dtype, post):
    """The backward has no use for the second norm's bias: one that lies off a vector boundary, alone,
    leaves the backward with the kernels for aligned tensors."""
    g = torch.Generator().manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    t = dict.fromkeys(R.NAMES)
    t.update(input=rn(70, 640), residual=rn(70, 640), weight=rn(640), bias=rn(641)[1:])
    if post:
        t.update(post_weight=rn(640), post_bias=rn(640))
    dy, ds = rn(70, 640), rn(70, 640)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    assert leaves["bias"].data_ptr() % 16
    want = R.nga_bounds({k: None if v is None else v.double() for k, v in t.items()}, dy.double(), ds.double(), dtype, post or "none",
                        "layernorm", "none", 1.0, 1.0, 0.0)
    y, s = fl.fused_norm_gate_add_norm(leaves["input"], leaves["residual"], None, leaves.get("post_weight"), leaves.get("post_bias"),
                                       leaves["weight"], leaves["bias"], post_norm=post, norm="layernorm", post_eps=R.EPS1,
                                       eps=R.EPS2)
    R.check(y.detach(), want["y"], "y"), R.check(s.detach(), want["sum"], "sum")
    for k, v in zip(leaves, torch.autograd.grad([y, s], list(leaves.values()), [dy, ds])):
        R.check(v, want["grads"][k], k)


WIDTHS = [(F32, 4356), (F32, 4608), (F32, 4864), (F32, 5056), (F32, 5120), (BF16, 5064), (F16, 4888), (BF16, 3584), (F16, 7168),
          (BF16, 6144), (F32, 1536), (BF16, 1528)]


@pytest.mark.parametrize("dtype,h", WIDTHS, ids=str)
@pytest.mark.parametrize("gate", ["none", "element"])
@pytest.mark.parametrize("norm", ["rmsnorm", "layernorm"])
def test_row_lengths_between_the_common_ones(dtype, h, gate, norm):
    """Row lengths around those at which the number of threads per row, or what stays in shared memory,
    changes, whole and not; with the residual and both gradients."""
    check(dtype, (2, 33, h), gate, norm, norm, residual=True)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("h", [32, 64, 128, 256, 512, 120, 72])
@pytest.mark.parametrize("gate", ["none", "vector", "element"])
@pytest.mark.parametrize("post", ["rmsnorm", "layernorm"])
def test_heads_without_a_second_norm(dtype, h, gate, post):
    """The norm of a head and its gate, forward and backward, over rows that leave row groups empty."""
    for rows in (1, 31, 700):
        check(dtype, (1, rows, h), gate, post, "none", residual=False)


def check(dtype, shape, gate, post, norm, residual):
    g = torch.Generator().manual_seed(shape[-1] + shape[-2])
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    h, bias, act = shape[-1], post == "layernorm", "none" if gate == "none" else "silu"
    t = dict.fromkeys(R.NAMES)
    t.update(input=rn(*shape), residual=rn(*shape) if residual else None, post_weight=rn(h), post_bias=rn(h) if bias else None,
             gate=None if gate == "none" else rn(*(shape if gate == "element" else (h,))))
    if norm != "none":
        t.update(weight=rn(h), bias=rn(h) if bias else None)
    dy, ds = rn(*shape) if norm != "none" else None, rn(*shape)
    d = lambda v: None if v is None else v.double()
    want = R.nga_bounds({k: d(v) for k, v in t.items()}, d(dy), d(ds), dtype, post, norm, act, 0.7, 1.0, 0.0)
    leaves = {k: v.detach().requires_grad_(True) for k, v in t.items() if v is not None}
    y, s = fl.fused_norm_gate_add_norm(*[leaves.get(n) for n in R.NAMES], post_norm=post, norm=norm, gate_activation=act,
                                       branch_scale=0.7, post_eps=R.EPS1, eps=R.EPS2)
    R.check(s.detach(), want["sum"], "sum")
    if y is not None:
        R.check(y.detach(), want["y"], "y")
    outs, gs = ([s], [ds]) if y is None else ([y, s], [dy, ds])
    for k, v in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs)):
        R.check(v, want["grads"][k], k)
