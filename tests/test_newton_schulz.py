"""Matrices orthogonalised by Newton-Schulz products and the update built on
them (mfx_newton_schulz, mfx_muon_update) against the formulas in 64 bits, and
their refusals.

Tolerances, of a result's norm.  Five steps are fifteen products.  In two terms
each operand is off by 2^-24 of its entries and a sum of up to 2^13 terms in fp32
by sqrt(2^13) 2^-24 < 2^-17 of the product's norm; fifteen of them that are not
aligned add up to four times that, and the iteration raises what falls on small
singular values against large ones, on average over a spectrum with a few large
values by up to four: 2^-13.  In one term an f16 operand is off by 2^-11 / sqrt(12) of
its norm, times the same sixteen: 2^-8.8, taken as 2^-8.  A result's own rounding is
at most half a step.  No entry is off by more than 32 times its share: sums of
many independent roundings, of which a matrix has under 2^24, stay within 6 of
their deviation, and the rows of a matrix with large directions within 5 of each
other."""
import ctypes

import numpy as np
import pytest

EPS = {"f32": 2.0 ** -23, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}
TOL = {1: 2.0 ** -8, 2: 2.0 ** -13}
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4
QUINTIC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def iterate(torch, u, steps=5, coeffs=QUINTIC, eps=1e-7):
    """The definition on the CPU in 64 bits, [batch, m, n]."""
    u = u.double().cpu()
    x = u / (u.flatten(1).norm(dim=1)[:, None, None] + eps)
    wide = x.shape[1] <= x.shape[2]
    for i in range(steps):
        a, b, c = (float(np.float32(v)) for v in (coeffs[i] if isinstance(coeffs[0], tuple) else coeffs))
        s = x @ x.mT if wide else x.mT @ x
        q = a * torch.eye(s.shape[1], dtype=s.dtype) + b * s + c * s @ s
        x = q @ x if wide else x @ q
    return x


def near(got, ref, tol, name):
    """Norm and entries of [batch, m, n], matrix by matrix."""
    got = got.double().cpu().reshape(ref.shape)
    for g, r in zip(got, ref):
        off, norm = g - r, float(r.norm())
        assert float(off.norm()) <= (tol + EPS[name] / 2) * norm
        rms = norm / r.numel() ** 0.5
        assert float((off.abs() - EPS[name] / 2 * r.abs()).max()) <= 32 * tol * rms


def gradient(torch, B, m, n, name, seed=0, low=2.0, size=1e-3):
    g = torch.Generator("cuda").manual_seed(seed)
    k = max(1, min(m, n) // 16)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = torch.matmul(mk(B, m, k), mk(B, k, n)) * (low / k ** 0.5) + mk(B, m, n)
    return (x * size).to(dt(torch, name))


def f32_error(torch, u, ref, steps=5, coeffs=QUINTIC, eps=1e-7):
    """Of the definition in plain f32 products on the GPU, of the norm (the largest of the matrices')."""
    u = u.double()
    x = (u / (u.flatten(1).norm(dim=1)[:, None, None] + eps)).float()
    wide = x.shape[1] <= x.shape[2]
    for i in range(steps):
        a, b, c = coeffs[i] if isinstance(coeffs[0], tuple) else coeffs
        t = x.mT.contiguous()
        s = torch.bmm(x, t) if wide else torch.bmm(t, x)
        q = b * s + c * torch.bmm(s, s)
        x = a * x + (torch.bmm(q, x) if wide else torch.bmm(x, q))
    off = (x.double().cpu() - ref).flatten(1).norm(dim=1) / ref.flatten(1).norm(dim=1)
    return float(off.max())


CASES = [
    # B, m, n, in, out, terms
    (1, 1, 1, "f32", "f32", 0),
    (2, 1, 9, "f32", "f32", 0),
    (1, 7, 1, "bf16", "bf16", 0),
    (3, 37, 100, "f32", "f32", 0),
    (1, 64, 64, "f16", "f16", 0),
    (1, 65, 63, "f32", "f32", 0),
    (2, 130, 257, "bf16", "bf16", 0),
    (1, 300, 301, "bf16", "bf16", 0),
    (1, 300, 301, "bf16", "f32", 0),
    (1, 513, 333, "f32", "bf16", 1),
    (5, 96, 520, "f16", "f32", 1),
    (1, 512, 2048, "f32", "f32", 0),
    (1, 1000, 520, "bf16", "bf16", 0),
    (1, 600, 5000, "f32", "f32", 0),     # a long k: few tiles, shared out
    (1, 5001, 258, "bf16", "bf16", 0),
    (2, 1100, 1300, "f32", "f32", 0),
    (1, 1543, 1537, "bf16", "bf16", 0),
    (12, 520, 264, "bf16", "bf16", 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=str)
def test_newton_schulz(cuda, nat, case):
    torch = cuda
    B, m, n, src, dst, terms = case
    g = gradient(torch, B, m, n, src)
    out = torch.full((B, m, n), float("nan"), device="cuda", dtype=dt(torch, dst))
    nat.newton_schulz(g, out=out, scale=0.75, terms=terms)
    one = terms == 1 or (terms == 0 and dst == "bf16" and min(m, n) >= 256)
    near(out, 0.75 * iterate(torch, g), TOL[1 if one else 2], dst)
    again = nat.newton_schulz(g, out_dtype=dt(torch, dst), scale=0.75, terms=terms)
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 4001, 4090), (1, 3490, 3400)], ids=str)
def test_large_sides(cuda, nat, shape):
    torch = cuda
    g = gradient(torch, *shape, "bf16", seed=4)
    near(nat.newton_schulz(g, steps=2, terms=1), iterate(torch, g, 2), TOL[1], "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 6])
@pytest.mark.parametrize("shape", [(1, 264, 8200), (1, 8193, 250), (3, 72, 4000)], ids=str)
def test_steps_of_long_matrices(cuda, nat, shape, steps):
    """Two steps at once, and the odd one behind them, each step with its own coefficients."""
    torch = cuda
    g = gradient(torch, *shape, "f32", seed=3)
    coeffs = [QUINTIC, (3.25, -4.5, 1.875), QUINTIC, (3.0, -4.0, 1.75), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)][:steps]
    out = nat.newton_schulz(g, steps=steps, coeffs=coeffs)
    near(out, iterate(torch, g, steps, coeffs), TOL[2], "f32")


@pytest.mark.gpu
def test_takes_singular_values_to_one(cuda, nat):
    """The cubic (1.5, -0.5, 0) repeated converges to U V^T of the singular value decomposition; its
    coefficients are exact and a small value s grows by 1.5 a step, at least 0.01 of |G| here: 24 steps."""
    torch = cuda
    for m, n in ((40, 90), (90, 40)):
        u, _, vt = np.linalg.svd(np.random.default_rng(1).standard_normal((m, n)), full_matrices=False)
        g = torch.from_numpy((u * np.linspace(0.1, 1.0, u.shape[1])) @ vt).float().cuda()
        out = nat.newton_schulz(g, steps=24, coeffs=(1.5, -0.5, 0.0))
        near(out, torch.from_numpy(u @ vt)[None], TOL[2], "f32")


@pytest.mark.gpu
def test_coefficients_of_each_step(cuda, nat):
    torch = cuda
    coeffs = [(4.0, -6.0, 2.5), (3.0, -3.5, 1.25), (1.875, -1.25, 0.375)]
    g = gradient(torch, 1, 100, 140, "f32", low=0.0)
    near(nat.newton_schulz(g, steps=3, coeffs=coeffs), iterate(torch, g, 3, coeffs), TOL[2], "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e25])
def test_any_size_of_gradient(cuda, nat, size):
    """Squares leave the range of fp32 on both sides; the result does not depend on the size (eps apart)."""
    torch = cuda
    g = gradient(torch, 1, 80, 120, "f32", size=size)
    near(nat.newton_schulz(g, eps=0.0), iterate(torch, g, eps=0.0), TOL[2], "f32")


@pytest.mark.gpu
def test_zeros_rank_and_values_that_are_not_finite(cuda, nat):
    """A matrix of zeros gives zeros, a singular one its definition, NaN and infinities stay in their matrix."""
    torch = cuda
    for m, n in ((70, 200), (200, 70)):
        g = gradient(torch, 6, m, n, "f32")
        g[1] = 0.0
        g[2, 3, 5] = float("nan")
        g[4, 0, 0] = float("inf")
        g[5] = g[5, :, :1] @ g[5, :1, :]
        out = nat.newton_schulz(g)
        ref = iterate(torch, g[[0, 1, 3, 5]])
        assert not out[1].any() and torch.isnan(out[2]).all() and torch.isnan(out[4]).any()
        near(out[[0, 3, 5]], ref[[0, 2, 3]], TOL[2], "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-42, 1e-37, 1e-34, 1e36, 1e37])
@pytest.mark.parametrize("shape", [(1, 80, 120), (2, 300, 70)], ids=str)
def test_sizes_at_the_ends_of_fp32(cuda, nat, shape, size):
    """Entries down to the smallest (of few bits: the reference takes them as they are) and up to the largest."""
    torch = cuda
    g = gradient(torch, *shape, "f32", size=size)
    assert torch.isfinite(g).all() and g.any()
    near(nat.newton_schulz(g, eps=0.0), iterate(torch, g, eps=0.0), TOL[2], "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-7, 1.2e-38, 2e-45])
def test_zeros_with_any_eps(cuda, nat, eps):
    """Zeros give zeros however small eps is, and weights that only decay."""
    torch = cuda
    z = torch.zeros(2, 70, 200, device="cuda")
    assert not nat.newton_schulz(z, eps=eps).any()  # (a NaN counts)
    for terms in (1, 2):
        assert not nat.newton_schulz(z.bfloat16().mT.contiguous(), eps=eps, terms=terms).any()
    w = torch.randn(2, 70, 200, device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    got, _ = nat.muon_update(w, z, z.clone(), lr=0.5, weight_decay=0.5, eps=eps, w_out=torch.empty_like(w))
    assert torch.equal(got, 0.75 * w)


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [100.0, 300.0])
@pytest.mark.parametrize("shape", [(1, 512, 512), (2, 300, 1000), (1, 2048, 264)], ids=str)
def test_one_direction_far_above_the_rest(cuda, nat, shape, ratio):
    """What the iteration raises by a^steps is what the operands' roundings leave of the rest, so a bf16
    result too needs products of f32.  Held to eight times the error of plain f32 products on the same
    matrix: an operand in two terms keeps 22 bits, four times f32's step, and the product of the second terms
    is left out, once more."""
    torch = cuda
    B, m, n = shape
    g = torch.Generator("cuda").manual_seed(6)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x = (mk(B, m, 1) * mk(B, 1, n) + mk(B, m, n) / ratio).bfloat16()
    ref = iterate(torch, x)
    tol = 8 * f32_error(torch, x, ref)
    near(nat.newton_schulz(x), ref, tol, "bf16")
    near(nat.newton_schulz(x, out_dtype=torch.float32), ref, tol, "f32")
    w, _ = nat.muon_update(torch.zeros_like(x), x, lr=-1.0)
    near(w, ref, tol, "bf16")
    f16 = x.half()
    near(nat.newton_schulz(f16), iterate(torch, f16), tol, "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("low", [2.0, 0.0])
@pytest.mark.parametrize("shape", [(1, 65, 63), (1, 250, 1000), (1, 1000, 520), (3, 2048, 512), (1, 600, 5000), (1, 5001, 258),
                                   (1, 1543, 1537), (1, 1100, 1301), (1, 2047, 4099), (1, 3500, 3333)], ids=str)
def test_two_terms_block_by_block(cuda, nat, shape, low):
    """No part of a result is worse than the rest: each block of 32 x 32 is held to eight times what plain f32
    products make of the matrix (four times f32's step in an operand, and the product left out once more), of
    the block's share of it or of its own norm, whichever is more."""
    torch = cuda
    B, m, n = shape
    g = gradient(torch, B, m, n, "f32", seed=11, low=low)
    ref = iterate(torch, g)
    tol = 8 * f32_error(torch, g, ref)
    off = nat.newton_schulz(g).double().cpu() - ref
    pad = (0, -n % 32, 0, -m % 32)

    def blocks(v):
        v = torch.nn.functional.pad(v, pad)
        return v.reshape(B, v.shape[1] // 32, 32, v.shape[2] // 32, 32).square().sum((2, 4)).sqrt()

    share = ref.flatten(1).norm(dim=1)[:, None, None] * 32 / (m * n) ** 0.5
    assert ((off.flatten(1).norm(dim=1) <= tol * ref.flatten(1).norm(dim=1))).all()
    assert (blocks(off) <= tol * torch.maximum(blocks(ref), share)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 300, 301), (1, 1000, 520), (1, 5001, 258), (1, 258, 4999), (1, 1543, 1537), (12, 520, 264),
                                   (1, 65, 63)], ids=str)
def test_one_term_where_asked_for(cuda, nat, shape):
    torch = cuda
    g = gradient(torch, *shape, "bf16", seed=9)
    near(nat.newton_schulz(g, terms=1), iterate(torch, g), TOL[1], "bf16")
    w, _ = nat.muon_update(torch.zeros_like(g), g, lr=-1.0, terms=1)
    assert torch.equal(w, nat.newton_schulz(g, terms=1))


@pytest.mark.gpu
def test_strided_and_in_place(cuda, nat):
    """Matrices inside wider ones at any alignment; out over g: the same bits."""
    torch = cuda
    for m, n, name in ((50, 131, "bf16"), (300, 270, "f32")):
        g = gradient(torch, 3, m, n, name)
        want = nat.newton_schulz(g)
        wide = torch.full((3, m + 2, n + 5), 7.0, device="cuda", dtype=g.dtype)
        wide[:, 1:1 + m, 3:3 + n] = g
        view = wide[:, 1:1 + m, 3:3 + n]
        assert nat.newton_schulz(view, out=view) is view
        assert torch.equal(view, want)
        assert (wide[:, 0] == 7).all() and (wide[:, -1] == 7).all() and (wide[..., :3] == 7).all() and (wide[..., 3 + n:] == 7).all()
        assert torch.equal(nat.newton_schulz(g[1]), want[1])


MUON = [
    # B, m, n, weights, gradient, momentum, nesterov, terms
    (1, 200, 300, "f32", "f32", "f32", True, 0),
    (2, 300, 130, "f32", "bf16", "f32", False, 0),
    (1, 300, 520, "bf16", "bf16", "bf16", True, 0),
    (1, 520, 259, "f16", "f16", "f32", True, 0),
    (3, 33, 65, "bf16", "f32", "bf16", False, 0),
    (1, 300, 301, "f32", "bf16", None, True, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", MUON, ids=str)
def test_muon_update(cuda, nat, case):
    torch = cuda
    B, m, n, wname, gname, bname, nesterov, terms = case
    lr, mu, decay, scale = 0.02, 0.9, 0.25, 3.0
    g = gradient(torch, B, m, n, gname)
    w = gradient(torch, B, m, n, wname, seed=1, low=0.0, size=0.05)
    buf = gradient(torch, B, m, n, bname, seed=2) if bname else None
    kw = dict(lr=lr, mu=mu, weight_decay=decay, scale=scale, nesterov=nesterov, terms=terms)
    f = lambda v: float(np.float32(v))  # noqa: E731
    u, new = g.double().cpu(), None
    if bname:
        new = f(mu) * buf.double().cpu() + (1 - f(mu)) * u
        u = f(mu) * new + (1 - f(mu)) * u if nesterov else new
    step = -f(lr) * f(scale) * iterate(torch, u)
    keep = (1 - f(lr) * f(decay)) * w.double().cpu()
    copies = w.clone(), None if buf is None else buf.clone()
    wo, bo = torch.empty_like(w), None if buf is None else torch.empty_like(buf)
    got_w, got_b = nat.muon_update(w, g, buf, w_out=wo, momentum_out=bo, **kw)
    assert got_w is wo and got_b is bo and torch.equal(w, copies[0]) and (buf is None or torch.equal(buf, copies[1]))
    one = terms == 1 or (terms == 0 and wname == "bf16" and min(m, n) >= 256)
    for k in range(B):
        off = (got_w[k].double().cpu() - (keep + step)[k]).abs() - EPS[wname] / 2 * (keep + step)[k].abs()
        share = TOL[1 if one else 2] * 32 * float(step[k].norm()) / (m * n) ** 0.5
        assert float((off - 4 * 2.0 ** -24 * keep[k].abs()).max()) <= share
    if bname:
        off = (got_b.double().cpu() - new).abs() - EPS[bname] / 2 * new.abs()
        mag = buf.double().cpu().abs() + g.double().cpu().abs()
        tiny = 2.0 ** -25 if bname == "f16" else 0.0
        assert float((off - 4 * 2.0 ** -24 * mag).max()) <= tiny
    # In place: the same bits.
    assert nat.muon_update(w, g, buf, **kw) == (w, buf) if buf is None else True
    if buf is not None:
        a, b = nat.muon_update(w, g, buf, **kw)
        assert a is w and b is buf and torch.equal(b, bo)
    assert torch.equal(w, wo)


@pytest.mark.gpu
def test_captured_and_on_two_streams(cuda, nat):
    """A graph of in-place updates replayed with eager work between; two streams at once."""
    torch = cuda
    shape = (2, 300, 520)
    g, w, buf = (gradient(torch, *shape, "f32", seed=k) for k in range(3))
    ws = [w.clone(), buf.clone()]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        nat.muon_update(ws[0].clone(), g, ws[1].clone(), lr=0.1)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            nat.muon_update(ws[0], g, ws[1], lr=0.1)
            o = nat.newton_schulz(g, terms=1)
    for _ in range(3):
        g.copy_(torch.roll(g, 1, 2) * 1.5)
        graph.replay()
        torch.cuda.synchronize()
        nat.muon_update(w, g, buf, lr=0.1)
        assert torch.equal(w, ws[0]) and torch.equal(buf, ws[1]) and torch.equal(o, nat.newton_schulz(g, terms=1))
    other = gradient(torch, 1, 700, 90, "bf16", seed=7)
    want = [nat.newton_schulz(x) for x in (g, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, x in enumerate((g, other)):
            with torch.cuda.stream(streams[k]):
                got[k].append(nat.newton_schulz(x))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[k]) for k in range(2) for x in got[k])


@pytest.mark.gpu
def test_no_matrices(cuda, nat):
    torch = cuda
    x = torch.empty(0, 5, 6, device="cuda")
    assert nat.newton_schulz(x).shape == (0, 5, 6)
    w, b = nat.muon_update(x, x, x.clone(), lr=0.1)
    assert w is x and b.shape == (0, 5, 6)


def _fill(nat, a, **kw):
    for i, f in enumerate(("g", "out", "w", "w_out", "momentum", "momentum_out")):
        if hasattr(a, f):
            setattr(a, f, 0x100000 * (i + 1))
    a.batch, a.m, a.n, a.steps, a.num_coeffs, a.eps, a.scale = 2, 64, 96, 5, 1, 1e-7, 1.0
    a.keep = (ctypes.c_float * 3)(*kw.pop("coeffs3", QUINTIC))
    a.coeffs = ctypes.addressof(a.keep)
    for f, _ in a._fields_:
        if f.endswith("row_stride"):
            setattr(a, f, 96)
        if f.endswith("batch_stride"):
            setattr(a, f, 64 * 96)
    if hasattr(a, "lr"):
        a.lr, a.mu = 0.1, 0.9
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_refusals(nat):
    lib = nat.load()

    def ns(**kw):
        a = _fill(nat, nat.NewtonSchulzArgs(), **kw)
        assert lib.mfx_newton_schulz_workspace_size(ctypes.byref(a)) == 0 or "workspace" in kw
        return lib.mfx_newton_schulz(ctypes.byref(a), None)

    def muon(**kw):
        a = _fill(nat, nat.MuonUpdateArgs(), **kw)
        assert lib.mfx_muon_update_workspace_size(ctypes.byref(a)) == 0 or "workspace" in kw
        return lib.mfx_muon_update(ctypes.byref(a), None)

    nan = float("nan")
    for call in (ns, muon):
        for bad in (dict(batch=-1), dict(m=0), dict(n=0), dict(steps=0), dict(coeffs=0), dict(num_coeffs=2), dict(eps=nan),
                    dict(eps=-1.0), dict(scale=nan), dict(terms=3), dict(terms=-1), dict(g=0), dict(g=0x100001),
                    dict(g_row_stride=-1), dict(coeffs3=(nan, 0, 0))):
            assert call(**bad) == INVALID, bad
        for bad in (dict(steps=33), dict(dtype=3), dict(m=2 ** 20 + 1, n=8), dict(m=2 ** 20, n=2 ** 20), dict(batch=65536),
                    dict(coeffs3=(30.0, 0.0, 0.0)), dict(coeffs3=(3.4445, -4.775, 60.0))):
            assert call(**bad) == UNSUPPORTED, bad
        assert call(workspace=0x900000, workspace_bytes=64) == WORKSPACE
        assert call(workspace=0x900001, workspace_bytes=1 << 30) == INVALID
    for bad in (dict(out=0), dict(out_row_stride=95), dict(out_batch_stride=63 * 96)):
        assert ns(**bad) == INVALID, bad
    assert ns(out_dtype=9) == UNSUPPORTED
    for bad in (dict(w=0), dict(w_out=0), dict(momentum=0), dict(momentum_out=0), dict(w_out_row_stride=95),
                dict(momentum_out_batch_stride=95), dict(lr=nan), dict(mu=1.5), dict(mu=nan), dict(weight_decay=float("inf"))):
        assert muon(**bad) == INVALID, bad
    assert muon(w_dtype=4) == muon(momentum_dtype=4) == UNSUPPORTED


def test_python_checks(nat):
    torch = pytest.importorskip("torch")
    x = torch.zeros(4, 6)
    for call in (lambda: nat.newton_schulz(x[0]), lambda: nat.newton_schulz(x, out=torch.zeros(6, 4)),
                 lambda: nat.newton_schulz(x.t()), lambda: nat.newton_schulz(x, coeffs=(1.0, 2.0)),
                 lambda: nat.newton_schulz(x, steps=3, coeffs=[(1.0, 2.0, 3.0)] * 2), lambda: nat.newton_schulz(x),
                 lambda: nat.muon_update(x, torch.zeros(4, 5), lr=0.1), lambda: nat.muon_update(x, x, x[:3], lr=0.1),
                 lambda: nat.muon_update(x, x, lr=0.1, momentum_out=x), lambda: nat.muon_update(x, x, lr=0.1, w_out=x.half())):
        with pytest.raises(ValueError):
            call()
