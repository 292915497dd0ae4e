"""Query / key norm with rotation (mfx_qk_norm_rope, mfx_qk_norm_rope_bwd)
against the formulas in 64 bits or more, and its refusals.

Tolerances.  Output element y from the pair (a, b): the kernel works in fp32
and rounds once, so |err| <= eps(dtype)/2 |y| for the rounding plus the fp32
steps before it -- the sum of squares (at most 22 adds deep, halved by the
root), root, division, two weight products, a sine and cosine within 2 steps,
two products and an add: under 32 half steps of |a| + |b|.  The backward's
terms r u w and r xh mean(u w xh) pass about twice as many: 64 half steps.  A
weight's gradient adds N products in fp32, at most N deep: (N + 64) half steps
of the sum of their magnitudes."""
import ctypes

import numpy as np
import pytest

HALF = 2.0 ** -24  # half a step of fp32
EPS = {"f32": 2.0 ** -23, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def angles(pos, rot, theta, sections, inv_freq=None):
    """cos, sin [T, rot/2] of pos [A, T] in extended precision."""
    i = np.arange(rot // 2)
    f = (np.longdouble(theta) ** (-2 * np.longdouble(1) * i / rot) if inv_freq is None
         else np.asarray(inv_freq, np.longdouble))
    axis = np.repeat(np.arange(len(sections)), sections)
    ang = pos[axis].T.astype(np.longdouble) * f
    return np.cos(ang).astype(np.float64), np.sin(ang).astype(np.float64)


def pairs(x, rot, il):
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if il else (x[..., :rot // 2], x[..., rot // 2:rot])


def unpairs(a, b, x, rot, il):
    out = x.copy()
    if il:
        out[..., 0:rot:2], out[..., 1:rot:2] = a, b
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = a, b
    return out


def forward(x, w, cos, sin, rot, il, eps):
    """(y, |a| + |b| of each output's pair); x [T, H, D], cos [T, rot/2]."""
    y = x.copy()
    if eps is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            y = y * w
    a, b = pairs(y, rot, il)
    c, s = cos[:, None], sin[:, None]
    mag = unpairs(abs(a) + abs(b), abs(a) + abs(b), abs(y), rot, il)
    return unpairs(a * c - b * s, b * c + a * s, y, rot, il), mag


def backward(x, w, g, cos, sin, rot, il, eps):
    """(dx, its terms' magnitude, dw, its terms' magnitude)."""
    c, s = cos[:, None], sin[:, None]
    a, b = pairs(g, rot, il)
    u = unpairs(a * c + b * s, b * c - a * s, g, rot, il)
    um = unpairs(abs(a) + abs(b), abs(a) + abs(b), abs(g), rot, il)
    if eps is None:
        return u, um, None, None
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * r
    ww = 1.0 if w is None else w
    gx, gm = u * ww, um * np.abs(ww)
    dx = r * (gx - xh * (gx * xh).mean(-1, keepdims=True))
    mag = r * (gm + abs(xh) * (gm * abs(xh)).mean(-1, keepdims=True))
    return dx, mag, (u * xh).sum((0, 1)), (um * abs(xh)).sum((0, 1))


def host(t):
    return t.double().cpu().numpy()


CASES = [
    # dtype, T, Hq, Hkv, D, rot, sections, interleaved, param dtype, eps
    ("bf16", 5, 4, 2, 128, 128, [64], False, "bf16", 1e-6),
    ("bf16", 300, 32, 8, 128, 128, [64], False, "f32", 1e-6),
    ("f16", 37, 6, 3, 96, 96, [8, 20, 20], True, "f32", 1e-5),
    ("f32", 1, 8, 8, 64, 64, [32], False, "f32", 1e-6),
    ("f32", 129, 3, 1, 256, 256, [64, 64], False, "f32", 0.0),
    ("bf16", 7, 5, 1, 80, 40, [20], False, "bf16", 1e-6),   # half the head turned, chunks of 4
    ("f16", 9, 3, 3, 64, 32, [3, 4, 4, 5], True, "f16", 1e-6),
    ("f32", 11, 2, 2, 33, 10, [5], False, "f32", 1e-6),     # an odd head: single elements
    ("bf16", 4, 2, 1, 255, 254, [127], True, "f32", 1e-6),  # two units a lane
    ("bf16", 6, 4, 4, 128, 0, [0], False, "bf16", 1e-6),    # norm alone
    ("f32", 6, 4, 2, 64, 64, [32], True, None, 1e-6),       # no weights
    ("bf16", 6, 4, 2, 64, 64, [0, 32], False, None, None),  # rotation alone; an axis without pairs
    ("f16", 3, 1, 1, 2, 2, [1], False, "f32", 1e-6),
    ("f32", 2, 1, 1, 1, 0, [0], False, "f32", 1e-6),
]


def make(torch, case, seed=0, far=1 << 20):
    name, T, Hq, Hkv, D, rot, sections, il, pname, eps = case
    rng = np.random.default_rng(seed)
    mk = lambda *s: torch.from_numpy(rng.standard_normal(s)).to(dt(torch, name)).cuda()  # noqa: E731
    q, k, gq, gk = mk(T, Hq, D), mk(T, Hkv, D), mk(T, Hq, D), mk(T, Hkv, D)
    w = [None, None]
    if pname:
        w = [torch.from_numpy(1 + 0.3 * rng.standard_normal(D)).to(dt(torch, pname)).cuda() for _ in range(2)]
    pos = rng.integers(-far, far, (len(sections), T)).astype(np.int32)
    return q, k, gq, gk, w, pos


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=[f"{c[0]}-T{c[1]}-D{c[4]}-rot{c[5]}" for c in CASES])
def test_forward_and_backward(cuda, nat, case):
    torch = cuda
    name, T, Hq, Hkv, D, rot, sections, il, pname, eps = case
    q, k, gq, gk, w, pos = make(torch, case)
    table = nat.rope_table(rot, 10000.0) if rot else None
    cos, sin = angles(pos, rot, 10000.0, sections)
    kw = dict(q_weight=w[0], k_weight=w[1], eps=eps, sections=sections, interleaved=il)
    if not rot:
        kw.pop("sections")
    pd = torch.from_numpy(pos).cuda()
    outs = nat.qk_norm_rope(q, k, pd, table, **kw)
    grads = nat.qk_norm_rope_bwd(q, k, gq, gk, pd, table, **kw)
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        wi = host(w[i]) if w[i] is not None else None
        ref, mag = forward(host(x), wi, cos, sin, rot, il, eps)
        assert (abs(host(outs[i]) - ref) <= EPS[name] / 2 * abs(ref) + 32 * HALF * mag + TINY[name]).all()
        dx, mag, dw, wmag = backward(host(x), wi, host(g), cos, sin, rot, il, eps)
        assert (abs(host(grads[i]) - dx) <= EPS[name] / 2 * abs(dx) + 64 * HALF * mag + TINY[name]).all()
        if w[i] is None:
            assert grads[2 + i] is None
            continue
        n = x.shape[0] * x.shape[1]
        got = grads[2 + i]
        assert got.dtype == w[i].dtype
        assert (abs(host(got) - dw) <= EPS[pname] / 2 * abs(dw) + (n + 64) * HALF * wmag + TINY[pname]).all()


@pytest.mark.gpu
def test_positions_of_any_size_keep_their_angle(cuda, nat):
    """32-bit positions up to their ends: the angle is exact modulo a turn."""
    torch = cuda
    pos = np.array([[-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 2, 10 ** 9 + 7, -1, 0, 1, 2 ** 24 + 1]], np.int32)
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((8, 2, 64))).float().cuda()
    inv = rng.uniform(-7, 7, 32)  # also past a turn a position, and backwards
    table = nat.rope_table(64, inv_freq=inv)
    y, _ = nat.qk_norm_rope(x, None, torch.from_numpy(pos[0]).cuda(), table, eps=None)
    # 64-bit frequencies times 2^31 are beyond extended precision's 2 pi: reduce exactly.
    from fractions import Fraction

    pi2 = Fraction(2) * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    ang = np.array([[float((Fraction(int(p)) * Fraction(float(f))) % pi2) for f in inv] for p in pos[0]])
    ref, mag = forward(x.double().cpu().numpy(), None, np.cos(ang), np.sin(ang), 64, False, None)
    # The frequency as the table holds it (extended precision over 2 pi, then
    # 2^-65 turns) moves the farthest angle by under 2 pi 2^31 (2^-64 + 2^-65).
    extra = 2 * np.pi * 2.0 ** 31 * 1.5 * 2.0 ** -63
    assert (abs(y.double().cpu().numpy() - ref) <= (32 * HALF + extra) * mag).all()


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["bhtd", "bthd"])
def test_layouts_strides_and_in_place(cuda, nat, layout):
    """4-D layouts, slices of one projection, positions per batch, outputs in
    a strided cache, in place: bit for bit the packed call's rows."""
    torch = cuda
    B, T, Hq, Hkv, D = 3, 17, 6, 2, 64
    g = torch.Generator("cuda").manual_seed(5)
    qkv = torch.randn(B, T, Hq + 2 * Hkv, D, device="cuda", generator=g).bfloat16()
    q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv]
    pos = torch.randint(0, 5000, (B, T), device="cuda", generator=g, dtype=torch.int32)
    w = torch.rand(D, device="cuda", generator=g) + 0.5
    table = nat.rope_table(D)
    kw = dict(q_weight=w, k_weight=w)
    want_q, want_k = nat.qk_norm_rope(q.reshape(B * T, Hq, D), k.reshape(B * T, Hkv, D), pos.reshape(-1), table, **kw)
    want_q, want_k = want_q.view(B, T, Hq, D), want_k.view(B, T, Hkv, D)
    turn = (lambda x: x.transpose(1, 2)) if layout == "bhtd" else (lambda x: x)
    cache = torch.full((B, Hkv, 40, D), 7.0, device="cuda", dtype=torch.bfloat16)
    view = cache[:, :, 5:5 + T]
    oq, ok = nat.qk_norm_rope(turn(q), turn(k), pos, table, layout=layout,
                              k_out=view if layout == "bhtd" else view.transpose(1, 2), **kw)
    assert torch.equal(oq, turn(want_q)) and torch.equal(view, want_k.transpose(1, 2))
    assert (cache[:, :, :5] == 7).all() and (cache[:, :, 5 + T:] == 7).all()
    # Positions shared by the batch (stride 0), keys alone, then in place.
    one, none = nat.qk_norm_rope(None, turn(k), pos[0], table, k_weight=w, layout=layout)[::-1]
    assert none is None
    many, _ = nat.qk_norm_rope(turn(k), None, pos[0].expand(B, T), table, q_weight=w, layout=layout)
    assert torch.equal(one, many)
    v_before = qkv[:, :, Hq + Hkv:].clone()
    nat.qk_norm_rope(turn(q), turn(k), pos, table, layout=layout, q_out=turn(q), k_out=turn(k), **kw)
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(qkv[:, :, Hq + Hkv:], v_before)


@pytest.mark.gpu
def test_unaligned_rows(cuda, nat):
    """Rows off 16 bytes take narrower chunks and give the same values."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(6)
    table = nat.rope_table(64)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    for off, stride in ((1, 65), (4, 68), (0, 66)):
        buf = torch.randn(off + 9 * 3 * stride, device="cuda", generator=g).half()
        x = buf[off:].as_strided((9, 3, 64), (3 * stride, stride, 1), off)
        a, _ = nat.qk_norm_rope(x, None, pos, table)
        b, _ = nat.qk_norm_rope(x.contiguous(), None, pos, table)
        # (The sum of squares is folded over other lanes: a rounding may differ.)
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -10 * b.float().abs().max()


@pytest.mark.gpu
def test_empty_rows_and_bad_values_stay_in_their_row(cuda, nat):
    torch = cuda
    table = nat.rope_table(64)
    x = torch.randn(5, 2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    pos = torch.arange(5, device="cuda", dtype=torch.int32)
    want = nat.qk_norm_rope(x, x, pos, table, q_weight=w, k_weight=w)
    y = x.clone()
    y[2, 1, 7] = float("nan")
    y[4, 0] = float("inf")
    got = nat.qk_norm_rope(y, y, pos, table, q_weight=w, k_weight=w)
    keep = torch.ones(5, 2, dtype=torch.bool)
    keep[2, 1] = keep[4, 0] = False
    for a, b in zip(want, got):
        assert torch.equal(a[keep], b[keep]) and b[2, 1].isnan().all() and not b[4, 0].isfinite().any()
    # A zero row stays zero (eps holds the root away from 0).
    z, _ = nat.qk_norm_rope(torch.zeros(1, 1, 64, device="cuda"), None, pos[:1], table)
    assert (z == 0).all()
    # No tokens: empty outputs, weight gradients of empty sums.
    e = x[:0]
    q, k = nat.qk_norm_rope(e, e, pos[:0], table, q_weight=w, k_weight=w)
    assert q.shape == (0, 2, 64) and k.shape == (0, 2, 64)
    _, _, dqw, dkw = nat.qk_norm_rope_bwd(e, e, e, e, pos[:0], table, q_weight=w, k_weight=w)
    assert (dqw == 0).all() and (dkw == 0).all()


@pytest.mark.gpu
def test_gradient_against_differences(cuda, nat):
    """f32 gradients against central differences of the kernel's own forward
    in the direction of the gradient."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(8)
    T, H, D = 6, 3, 64
    x, gy = (torch.randn(T, H, D, device="cuda", generator=g) for _ in range(2))
    w = torch.rand(D, device="cuda", generator=g) + 0.5
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    table = nat.rope_table(D)
    dx, _, dw, _ = nat.qk_norm_rope_bwd(x, None, gy, None, pos, table, q_weight=w)

    def f(x, w):
        return float((nat.qk_norm_rope(x, None, pos, table, q_weight=w)[0].double() * gy.double()).sum())

    h = 2.0 ** -8
    for d, args in ((dx, lambda e: (x + e * dx / dx.norm(), w)), (dw, lambda e: (x, w + e * dw / dw.norm()))):
        num = (f(*args(h)) - f(*args(-h))) / (2 * h)
        # Differences: outputs of size ~1 rounded to 2^-24, T H D of them at
        # random, over 2h; and the third derivative's h^2 / 6, below h^2.
        tol = 2.0 ** -23 * (T * H * D) ** 0.5 * 4 / (2 * h) + h * h * float(d.norm())
        assert abs(num - float(d.norm())) <= tol


@pytest.mark.gpu
def test_captured_backward_replays_with_new_inputs(cuda, nat):
    torch = cuda
    g = torch.Generator("cuda").manual_seed(9)
    T, Hq, Hkv, D = 70, 8, 2, 128
    mk = lambda h: torch.randn(T, h, D, device="cuda", generator=g).bfloat16()  # noqa: E731
    q, k, gq, gk = mk(Hq), mk(Hkv), mk(Hq), mk(Hkv)
    w = torch.ones(D, device="cuda")
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    table = nat.rope_table(D)
    run = lambda: nat.qk_norm_rope_bwd(q, k, gq, gk, pos, table, q_weight=w, k_weight=w)  # noqa: E731
    run()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run()
    for _ in range(3):
        for t in (q, k, gq, gk):
            t.copy_(torch.randn(t.shape, device="cuda", generator=g))
        pos.add_(13)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


# ---- refusals (no GPU needed) ----------------------------------------------------

def _args(nat, bwd=False, **over):
    """Argument struct of a valid bf16 call with made-up addresses."""
    a = (nat.QkNormRopeBwdArgs if bwd else nat.QkNormRopeArgs)()
    names = ("q", "k", "dq_out", "dk_out", "dq", "dk") if bwd else ("q", "k", "q_out", "k_out")
    for i, n in enumerate(names):
        setattr(a, n, 0x10000 * (i + 1))
    a.positions, a.freqs = 0x900000, 0xA00000
    a.B, a.T, a.Hq, a.Hkv, a.D, a.rot = 1, 4, 4, 2, 64, 64
    for n, _ in a._fields_:
        if n.endswith("_strides") and n != "pos_strides":
            h = 2 if n.startswith(("k", "dk")) else 4
            getattr(a, n)[:] = [4 * h * 64, 64, h * 64, 1]
    a.pos_strides[:] = [0, 0, 1]
    a.sections[:] = [32, 0, 0, 0]
    a.axes, a.dtype, a.param_dtype, a.eps = 1, nat.MFX_BF16, nat.MFX_BF16, 1e-6
    for n, v in over.items():
        if isinstance(v, list):
            getattr(a, n)[:len(v)] = v
        else:
            setattr(a, n, v)
    return a


BAD = [dict(q=0), dict(k=0), dict(D=0), dict(D=257, rot=0, sections=[0]), dict(rot=63), dict(rot=66), dict(rot=-2),
       dict(positions=0), dict(freqs=0), dict(axes=0), dict(axes=5), dict(sections=[31]), dict(sections=[-1, 33], axes=2),
       dict(eps=float("nan")), dict(eps=float("inf")), dict(eps=-1.0, q_weight=0x40), dict(dtype=9),
       dict(q_weight=0x40, param_dtype=2), dict(T=-1), dict(Hq=0, Hkv=0), dict(q_strides=[1024, 64, 256, 2]),
       dict(k_strides=[1024, 64, 256, 0]), dict(T=1 << 32), dict(B=1 << 16, T=1 << 16)]


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("over", BAD, ids=[",".join(o) for o in BAD])
def test_refuses(nat, bwd, over):
    lib = nat.load()
    a = _args(nat, bwd, **over)
    rc = (lib.mfx_qk_norm_rope_bwd if bwd else lib.mfx_qk_norm_rope)(ctypes.byref(a), None)
    assert rc in (-1, -2) and lib.mfx_last_error()
    if bwd:
        assert lib.mfx_qk_norm_rope_bwd_workspace_size(ctypes.byref(a)) == 0


def test_refuses_null_args_and_small_workspace(nat):
    lib = nat.load()
    assert lib.mfx_qk_norm_rope(None, None) == -1 and lib.mfx_qk_norm_rope_bwd(None, None) == -1
    assert lib.mfx_qk_norm_rope_bwd_workspace_size(None) == 0
    a = _args(nat, True, q_weight=0x40, dq_weight=0x80, workspace=0x100000, workspace_bytes=8)
    assert lib.mfx_qk_norm_rope_bwd_workspace_size(ctypes.byref(a)) >= 2 * 64 * 4
    assert lib.mfx_qk_norm_rope_bwd(ctypes.byref(a), None) == -4


def test_rope_freqs(nat):
    import torch

    t = nat.rope_table(8, 10000.0, device="cpu").numpy().view(np.uint64)
    want = [int(round(10000.0 ** (-2 * i / 8) / (2 * np.pi) * 2.0 ** 64)) for i in range(4)]
    assert all(abs(int(a) - b) <= 2 ** 13 for a, b in zip(t, want))  # (the check itself is in doubles)
    neg = nat.rope_table(4, inv_freq=[-1.0, 2 * np.pi + 0.5], device="cpu").numpy().view(np.uint64)
    assert abs(int(neg[0]) - (2 ** 64 - want[0])) <= 2 ** 13
    assert abs(int(neg[1]) / 2 ** 64 - 0.5 / (2 * np.pi)) < 1e-15
    for bad in (dict(rot=7), dict(rot=8, theta=0.0), dict(rot=8, theta=float("inf"))):
        with pytest.raises(nat.MfxError):
            nat.rope_table(**bad, device="cpu")
    with pytest.raises(ValueError):
        nat.rope_table(8, inv_freq=torch.ones(3), device="cpu")
    with pytest.raises(nat.MfxError):
        nat.rope_table(4, inv_freq=[1.0, float("nan")], device="cpu")


def test_wrapper_refuses(nat):
    import torch

    q, k = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64)
    pos, table = torch.zeros(4, dtype=torch.int32), nat.rope_table(64, device="cpu")
    for kw, err in ((dict(), ValueError), (dict(q=None, k=None), ValueError),
                    (dict(positions=pos.long()), TypeError), (dict(positions=pos[:3]), ValueError),
                    (dict(k=torch.zeros(5, 2, 64)), ValueError), (dict(k=k.half()), ValueError),
                    (dict(q_weight=torch.ones(63)), ValueError), (dict(sections=[32]), ValueError),
                    (dict(q=q.int(), k=None), TypeError)):
        args = dict(q=q, k=k, positions=pos, table=table, **{})
        args.update(kw)
        with pytest.raises(err):  # (the first: host tensors)
            nat.qk_norm_rope(**args)
