"""Cross entropy of a linear head (mfx_linear_xent, mfx_linear_xent_bwd)
against the formulas in 64 bits, and its refusals.

Tolerances.  A logit is a sum of H products in fp32: off by at most
(H + 2) 2^-24 of the sum of their magnitudes, and a row's lse by at most the
largest such error of its logits, plus the exponentials' and logarithm's steps,
2^-20 and 2^-22 of |lse|.  The loss adds the target's logit: twice that.
d = (p - onehot) g: p is off by twice a logit's error relative (its own and
lse's) and by 2^-20, and flushed to 0 below 2^-126; 16 bits then round d by eps/2, f16 besides by 2^-25 of the
power of two above the largest g.  dh and dw are sums of d times w or h: those
errors times the magnitudes, their own fp32 sums of n terms, (n + 4) 2^-24, and
the output's rounding, eps/2."""
import ctypes

import numpy as np
import pytest

EPS = {"f32": 2.0 ** -24, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def make(torch, name, T, H, V, seed=0, lift=8.0, target_dtype="int64"):
    g = torch.Generator("cuda").manual_seed(seed)
    w = (torch.randn(V, H, device="cuda", generator=g) * H ** -0.5).to(dt(torch, name))
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    wt = w[t].float()
    h = torch.randn(T, H, device="cuda", generator=g)
    h = (h + lift * torch.rand(T, 1, device="cuda", generator=g) * wt / (wt * wt).sum(1, keepdim=True)).to(dt(torch, name))
    if T > 3:
        t[T // 2] = -100
        t[T // 3] = V
    dloss = torch.rand(T, device="cuda", generator=g) / T
    return h, w, t.to(getattr(torch, target_dtype)), dloss


def check_all(torch, nat, name, h, w, t, dloss, dw_dtype=None):
    """Loss, lse and both gradients of one call each, against 64 bits."""
    T, H = h.shape
    V = w.shape[0]
    hd, wd, gd = h.double(), w.double(), dloss.double()
    z = hd @ wd.T
    zerr = (H + 2) * 2.0 ** -24 * (hd.abs() @ wd.abs().T)
    lse = torch.logsumexp(z, 1)
    counts = (t >= 0) & (t < V)
    tt = t.long().clamp(0, V - 1)[:, None]
    loss = torch.where(counts, lse - z.gather(1, tt)[:, 0], 0.0)
    err = zerr.amax(1) + 2.0 ** -20 + 2.0 ** -22 * lse.abs()
    loss_k, lse_k = nat.linear_xent(h, w, t)
    assert ((lse_k.double() - lse).abs() <= err).all()
    assert ((loss_k.double() - loss).abs() <= 2 * err).all() and (loss_k[~counts] == 0).all()

    g = torch.where(counts, gd, 0.0)[:, None]
    p = torch.exp(z - lse[:, None])
    d = p.clone()
    d.scatter_add_(1, tt, torch.full_like(d[:, :1], -1.0))
    d *= g
    e = EPS[name]
    derr = g.abs() * p * (zerr + err[:, None] + 2.0 ** -20) + (e / 2 if name != "f32" else 2.0 ** -23) * d.abs()
    derr = derr + g.abs() * 2.0 ** -126
    if name == "f16" and T:
        derr = derr + 2.0 ** -40 * g.abs().max()
    derr = derr + 2.0 ** -22 * d.abs()
    dh_k, dw_k = nat.linear_xent_bwd(h, w, t, lse_k, dloss, dw_dtype=dw_dtype)
    for got, ref, mag, dev in ((dh_k, d @ wd, d.abs() @ wd.abs(), derr @ wd.abs()),
                               (dw_k, d.T @ hd, d.abs().T @ hd.abs(), derr.T @ hd.abs())):
        n = V if got is dh_k else T
        oe = 2.0 ** -23 if got.dtype == torch.float32 else e
        tol = dev + (n + 4) * 2.0 ** -24 * (mag + dev) + oe / 2 * (ref.abs() + dev) + TINY[name]
        bad = (got.double() - ref).abs() > tol
        assert not bad.any(), (got.shape, bad.nonzero()[:3], ((got.double() - ref).abs() / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,H,V", [(1, 8, 1), (1, 64, 1000), (3, 8, 129), (33, 72, 257), (128, 128, 128), (130, 200, 511),
                                   (257, 512, 1000), (65, 64, 5000), (600, 136, 700), (1000, 64, 255)])
def test_sizes(cuda, nat, name, T, H, V):
    check_all(cuda, nat, name, *make(cuda, name, T, H, V))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("T,H,V", [(4100, 128, 4097), (4096, 64, 4096), (300, 4104, 520), (2049, 2056, 2050)])
def test_wide_tiles_and_ranges(cuda, nat, name, T, H, V):
    """Enough tiles for the 256-wide kernel, ragged on every side; long k."""
    check_all(cuda, nat, name, *make(cuda, name, T, H, V, seed=2))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V", [(33, 1028, 8001), (100, 2052, 300), (1, 4, 33), (70, 132, 31), (700, 200, 1501),
                                   (2100, 256, 4001), (4093, 260, 4095)])
def test_f32_tile_forms(cuda, nat, T, H, V):
    """32 x 32 blocks, 64 x 64 and 128 x 128 tiles, ragged on every side."""
    check_all(cuda, nat, "f32", *make(cuda, "f32", T, H, V, seed=4))


@pytest.mark.gpu
def test_several_pieces(cuda, nat):
    """d beyond its budget: a vocabulary in pieces, dh added up over them.
    (Against the same call on column blocks small enough for one piece.)"""
    torch = cuda
    T, H, V = 70000, 64, 9000
    h, w, t, dloss = make(torch, "bf16", T, H, V, seed=3)
    assert T * V * 2 > 2 * (512 << 20)
    loss, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss, dw_dtype=torch.float32)
    dhr, dwr = torch.zeros(T, H, device="cuda", dtype=torch.float64), torch.zeros(V, H, device="cuda")
    for a in range(0, T, 7000):  # (rows apart: one piece each)
        s = slice(a, a + 7000)
        x, y = nat.linear_xent_bwd(h[s], w, t[s], lse[s], dloss[s], dw_dtype=torch.float32)
        dhr[s] = x.double()
        dwr += y
    # dh: one rounding to bf16 each (the sums differ by fp32's order); dw: fp32
    # sums of T terms in another order, of which |d h| adds up to under 1.
    assert ((dh.double() - dhr).abs() <= 2.0 ** -7 * dhr.abs() + 2.0 ** -24).all()
    mag = float((dw.abs().max() + 1.0) * T * 2.0 ** -24)
    assert float((dw - dwr).abs().max()) <= mag


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_more_classes_than_a_piece_has_columns(cuda, nat, name):
    check_all(cuda, nat, name, *make(cuda, name, 3, 8, (1 << 21) + 1001, seed=11))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_int32_targets_strides_and_parts(cuda, nat, name):
    torch = cuda
    h, w, t, dloss = make(torch, name, 200, 64, 300, seed=4, target_dtype="int32")
    check_all(torch, nat, name, h, w, t, dloss, dw_dtype=torch.float32)
    loss, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss)
    # Wider rows than H, batch dims, outputs in place of the caller's.
    hb, wb = torch.full((200, 96), 9.0, device="cuda", dtype=h.dtype), torch.full((300, 80), 9.0, device="cuda", dtype=h.dtype)
    hb[:, 16:80], wb[:, :64] = h, w
    loss2, lse2 = nat.linear_xent(hb[:, 16:80], wb[:, :64], t)
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2)
    oh, ow = torch.full_like(hb, 5.0), torch.full_like(wb, 5.0)
    nat.linear_xent_bwd(hb[:, 16:80], wb[:, :64], t, lse, dloss, dh=oh[:, 16:80], dw=ow[:, :64])
    assert torch.equal(oh[:, 16:80], dh) and (oh[:, :16] == 5).all() and (oh[:, 80:] == 5).all()
    assert torch.equal(ow[:, :64], dw) and (ow[:, 64:] == 5).all()
    loss3, _ = nat.linear_xent(h.view(4, 50, 64), w, t.view(4, 50))
    assert loss3.shape == (4, 50) and torch.equal(loss3.view(-1), loss)
    only, none = nat.linear_xent_bwd(h, w, t, lse, dloss, need_dw=False)
    assert none is None and torch.equal(only, dh)
    none, only = nat.linear_xent_bwd(h, w, t, lse, dloss, need_dh=False)
    assert none is None and torch.equal(only, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_rows_that_do_not_count(cuda, nat, name):
    """Whatever their dloss, lse or h hold; a NaN row stays in its row."""
    torch = cuda
    h, w, t, dloss = make(torch, name, 150, 64, 300, seed=5)
    t[::3] = -1
    loss, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss)
    assert (loss[::3] == 0).all() and (dh[::3] == 0).all()
    d2, l2 = dloss.clone(), lse.clone()
    d2[::3], l2[::3] = float("nan"), float("-inf")
    a, b = nat.linear_xent_bwd(h, w, t, l2, d2)
    assert torch.equal(a, dh) and torch.equal(b, dw)
    t[:] = -100
    loss, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss)
    assert (loss == 0).all() and (dh == 0).all() and (dw == 0).all() and lse.isfinite().all()
    h2 = h.clone()
    h2[7] = float("nan")
    t[:] = 5
    loss, lse = nat.linear_xent(h, w, t)
    loss2, lse2 = nat.linear_xent(h2, w, t)
    keep = torch.arange(150, device="cuda") != 7
    assert torch.equal(loss[keep], loss2[keep]) and loss2[7].isnan() and lse2[7].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_large_logits(cuda, nat, name):
    """Logits of hundreds: the running maximum keeps the sums finite."""
    torch = cuda
    h, w, t, dloss = make(torch, name, 64, 64, 500, seed=6)
    check_all(torch, nat, name, h * 100, w, t, dloss)


@pytest.mark.gpu
def test_small_gradients_survive_f16(cuda, nat):
    """dloss of 1e-7, below f16's steps times any probability: the held power
    of two keeps d's digits; dh and dw themselves are taken in range."""
    torch = cuda
    h, w, t, _ = make(torch, "f16", 256, 64, 300, seed=7)
    one = torch.full((256,), 2.0 ** -23, device="cuda")
    big = torch.full((256,), 1.0, device="cuda")
    _, lse = nat.linear_xent(h, w, t)
    _, dw = nat.linear_xent_bwd(h, w, t, lse, one, dw_dtype=torch.float32)
    _, ref = nat.linear_xent_bwd(h, w, t, lse, big, dw_dtype=torch.float32)
    assert torch.equal(dw * 2.0 ** 23, ref)


@pytest.mark.gpu
def test_no_rows(cuda, nat):
    torch = cuda
    h, w, t, dloss = make(torch, "bf16", 4, 64, 300)
    loss, lse = nat.linear_xent(h[:0], w, t[:0])
    assert loss.shape == (0,) and lse.shape == (0,)
    for dtype in (None, torch.float32):
        dh, dw = nat.linear_xent_bwd(h[:0], w, t[:0], lse, dloss[:0], dw_dtype=dtype, dw=None)
        assert dh.shape == (0, 64) and (dw == 0).all()


@pytest.mark.gpu
def test_gradient_against_differences(cuda, nat):
    torch = cuda
    h, w, t, dloss = make(torch, "f32", 40, 32, 200, seed=8)
    dloss = dloss * 40
    _, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss)

    def f(h, w):
        return float((nat.linear_xent(h, w, t)[0].double() * dloss.double()).sum())

    e = 2.0 ** -5
    for d, at in ((dh, lambda s: (h + s * dh / dh.norm(), w)), (dw, lambda s: (h, w + s * dw / dw.norm()))):
        num = (f(*at(e)) - f(*at(-e))) / (2 * e)
        # Losses off by 2^-19 at random over 2 e, 40 of them of weight below 1;
        # the third derivative of a log-sum-exp is under e^2 of the step's logits.
        tol = 2.0 ** -19 * 40 ** 0.5 * 2 / (2 * e) + e * e * float(d.norm())
        assert abs(num - float(d.norm())) <= tol


@pytest.mark.gpu
def test_captured_step_replays(cuda, nat):
    torch = cuda
    h, w, t, dloss = make(torch, "f16", 300, 64, 1000, seed=9)

    def step():
        loss, lse = nat.linear_xent(h, w, t)
        return (loss, lse, *nat.linear_xent_bwd(h, w, t, lse, dloss))

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    for k in range(3):
        h.mul_(0.9)
        t.copy_(torch.roll(t, 1))
        dloss.mul_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_streams_at_once(cuda, nat):
    """Workspaces come from the allocator of the calling stream."""
    torch = cuda
    h, w, t, dloss = make(torch, "bf16", 500, 128, 3000, seed=10)
    loss, lse = nat.linear_xent(h, w, t)
    want = nat.linear_xent_bwd(h, w, t, lse, dloss)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                lo, ls = nat.linear_xent(h, w, t)
                got.append((lo, ls, *nat.linear_xent_bwd(h, w, t, ls, dloss)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], loss) and torch.equal(g[1], lse)
        assert torch.equal(g[2], want[0]) and torch.equal(g[3], want[1])


# ---- refusals (no GPU needed) ----------------------------------------------------

def _args(nat, bwd, **over):
    a = (nat.LinearXentBwdArgs if bwd else nat.LinearXentArgs)()
    names = ("h", "w", "targets", "lse", "dloss", "dh", "dw") if bwd else ("h", "w", "targets", "loss", "lse")
    for i, n in enumerate(names):
        setattr(a, n, 0x100000 * (i + 1))
    a.T, a.H, a.V = 10, 64, 100
    for n, _ in a._fields_:
        if n.endswith("_stride"):
            setattr(a, n, 64)
    a.dtype, a.target_dtype = nat.MFX_BF16, nat.MFX_I64
    if bwd:
        a.dw_dtype = nat.MFX_BF16
    for n, v in over.items():
        setattr(a, n, v)
    return a


BAD = [dict(h=0), dict(w=0), dict(targets=0), dict(T=-1), dict(H=0), dict(V=0), dict(dtype=7), dict(target_dtype=0),
       dict(H=60), dict(h_stride=63), dict(w_stride=65), dict(h=0x100004), dict(w=0x100008), dict(T=1 << 31),
       dict(V=1 << 31), dict(H=1 << 31, h_stride=1 << 31), dict(w_stride=1 << 21), dict(T=1 << 30, V=1 << 30)]
BAD_BWD = [dict(lse=0), dict(dloss=0), dict(dh=0, dw=0), dict(dw_dtype=2), dict(dh_stride=32), dict(dw_stride=60),
           dict(dw=0x700004), dict(dh=0x600008)]


@pytest.mark.parametrize("bwd,over", [(b, o) for b in (False, True) for o in BAD] + [(True, o) for o in BAD_BWD]
                         + [(False, dict(loss=0))], ids=str)
def test_refuses(nat, bwd, over):
    lib = nat.load()
    fn = "mfx_linear_xent_bwd" if bwd else "mfx_linear_xent"
    a = _args(nat, bwd, **over)
    assert getattr(lib, fn)(ctypes.byref(a), None) in (-1, -2) and lib.mfx_last_error()
    assert getattr(lib, fn + "_workspace_size")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("bwd", [False, True])
def test_refuses_null_args_and_workspace(nat, bwd):
    lib = nat.load()
    fn = "mfx_linear_xent_bwd" if bwd else "mfx_linear_xent"
    assert getattr(lib, fn)(None, None) == -1 and getattr(lib, fn + "_workspace_size")(None) == 0
    need = getattr(lib, fn + "_workspace_size")(ctypes.byref(_args(nat, bwd)))
    assert need > 0
    a = _args(nat, bwd, workspace=0x10000000, workspace_bytes=need - 1)
    assert getattr(lib, fn)(ctypes.byref(a), None) == -4
    a = _args(nat, bwd, workspace=0x10000010, workspace_bytes=need)
    assert getattr(lib, fn)(ctypes.byref(a), None) == -1


def test_wrapper_refuses(nat):
    import torch

    h, w, t = torch.zeros(9, 64), torch.zeros(20, 64), torch.zeros(9, dtype=torch.int64)
    for args, err in (((h, w, t), ValueError), ((h, w[:, :32], t), ValueError), ((h, w.half(), t), ValueError),
                      ((h, w, t[:8]), ValueError), ((h, w, t.short()), TypeError), ((h, w.t().contiguous().t(), t), ValueError),
                      ((h.int(), w.int(), t), TypeError)):
        with pytest.raises(err):  # (the first: host tensors)
            nat.linear_xent(*args)
    with pytest.raises(ValueError):
        nat.linear_xent_bwd(h, w, t, torch.zeros(9), torch.zeros(9, dtype=torch.float64))
    with pytest.raises(ValueError):
        nat.linear_xent_bwd(h, w, t, torch.zeros(9), torch.zeros(9), dw=torch.zeros(19, 64))
