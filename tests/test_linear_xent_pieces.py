"""Gradients of the linear head's cross entropy where d takes several pieces
of the vocabulary and the sums run over many rows, entry by entry against 64
bits.

Tolerances as test_linear_xent.py derives them: a logit is off by
(H + 2) 2^-24 of its terms' magnitudes, lse by the largest of those and 2^-20 +
2^-22 |lse|, p by both relative and 2^-20; d = (p - onehot) g is rounded by
eps/2 in 16 bits (f16 also by 2^-40 of the largest g), its division by the largest
g and the product with it at the end by 2^-22; the sums' n fp32 steps are off by
(n + 4) 2^-24 of their terms' magnitudes and the result's rounding by eps/2.
All of it scales with the terms that an entry sums, so an entry of a piece that
is missing, doubled or another's is out of bounds (`test_bounds_catch`)."""
import pytest

from test_linear_xent import EPS, TINY, dt, make


def bounds(torch, name, h, w, t, dloss, block=4096):
    """(dh, its bound, dw, its bound) in 64 bits, rows in blocks; bounds without
    the results' own rounding."""
    (T, H), V = h.shape, w.shape[0]
    e = EPS[name]
    wd = w.double()
    dh, mh = torch.zeros(T, H, dtype=torch.float64, device=h.device), torch.zeros(T, H, dtype=torch.float64, device=h.device)
    dw, mw = torch.zeros_like(wd), torch.zeros_like(wd)
    top = float(dloss.abs().max())
    for a in range(0, T, block):
        s = slice(a, min(a + block, T))
        hd = h[s].double()
        z = hd @ wd.T
        zerr = (H + 2) * 2.0 ** -24 * (hd.abs() @ wd.abs().T)
        lse = torch.logsumexp(z, 1, keepdim=True)
        err = zerr.amax(1, keepdim=True) + 2.0 ** -20 + 2.0 ** -22 * lse.abs()
        tt = t[s].long()
        counts = ((tt >= 0) & (tt < V))[:, None]
        g = torch.where(counts, dloss[s].double()[:, None], 0.0)
        p = torch.exp(z - lse)
        d = p.clone()
        d.scatter_add_(1, tt.clamp(0, V - 1)[:, None], torch.full_like(g, -1.0))
        d *= g
        derr = g.abs() * p * (zerr + err + 2.0 ** -20) + (e / 2 if name != "f32" else 2.0 ** -23) * d.abs()
        derr += 2.0 ** -22 * d.abs() + g.abs() * 2.0 ** -126
        if name == "f16":
            derr += 2.0 ** -40 * top
        dh[s], dw = d @ wd, dw + d.T @ hd
        mh[s] = derr @ wd.abs() + (V + 4) * 2.0 ** -24 * ((d.abs() + derr) @ wd.abs())
        mw += derr.T @ hd.abs() + (T + 4) * 2.0 ** -24 * ((d.abs() + derr).T @ hd.abs())
    return dh, mh, dw, mw


def out_of_bounds(torch, name, got, ref, bound):
    """Entries off by more than the bound and the rounding of got's type."""
    oe = 2.0 ** -23 if got.dtype == torch.float32 else EPS[name]
    return (got.double() - ref).abs() > bound + oe / 2 * (ref.abs() + bound) + TINY[name]


@pytest.mark.gpu
@pytest.mark.parametrize("name,T,H,V,pieces", [("bf16", 70000, 64, 9000, 3), ("f16", 70000, 72, 8200, 3),
                                               ("f32", 40000, 36, 9001, 3), ("bf16", 270001, 8, 1300, 2)])
def test_pieces_and_many_rows(cuda, name, T, H, V, pieces):
    torch = cuda
    from jax_mlx_amd import native as nat

    size = torch.finfo(dt(torch, name)).bits // 8
    assert T * V * size > (pieces - 1) * (512 << 20)
    h, w, t, dloss = make(torch, name, T, H, V, seed=3)
    _, lse = nat.linear_xent(h, w, t)
    dh, dw = nat.linear_xent_bwd(h, w, t, lse, dloss, dw_dtype=torch.float32)
    rh, mh, rw, mw = bounds(torch, name, h, w, t, dloss)
    for what, got, ref, bound in (("dh", dh, rh, mh), ("dw", dw, rw, mw)):
        bad = out_of_bounds(torch, name, got, ref, bound)
        assert not bad.any(), (what, bad.nonzero()[:3], ((got.double() - ref).abs() / bound).max())
    # In the inputs' type: the same sums, rounded once more.
    _, dw = nat.linear_xent_bwd(h, w, t, lse, dloss, need_dh=False)
    assert not out_of_bounds(torch, name, dw, rw, mw).any()


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_bounds_catch(name):
    """Of the same recipe on the CPU: d rounded as the kernels round it stays in
    bounds; a piece left out, doubled or taken from its neighbour, a row
    weight of another row and a sum short of rows do not."""
    import torch

    gen = torch.Generator().manual_seed(3)
    T, H, V, piece = 2100, 64, 768, 256
    w = (torch.randn(V, H, generator=gen) * H ** -0.5).to(dt(torch, name))
    t = torch.randint(0, V, (T,), generator=gen)
    t[T // 2], t[T // 3] = -100, V
    h = torch.randn(T, H, generator=gen).to(dt(torch, name))
    dloss = torch.rand(T, generator=gen) / T
    rh, mh, rw, mw = bounds(torch, name, h, w, t, dloss, block=700)

    def grads(weight):
        z = h.double() @ w.double().T
        d = torch.softmax(z, 1)
        d[torch.arange(T), t.clamp(0, V - 1)] -= 1.0
        d = d * torch.where((t >= 0) & (t < V), weight.double(), 0.0)[:, None] / weight.max()
        d = d.to(dt(torch, name)).double() * weight.max()
        return (d @ w.double()).to(dt(torch, name)), (d.T @ h.double()).float()

    def bad(dh, dw):
        return (float(out_of_bounds(torch, name, dh, rh, mh).float().mean()),
                float(out_of_bounds(torch, name, dw, rw, mw).float().mean()))

    dh, dw = grads(dloss)
    assert bad(dh, dw) == (0.0, 0.0)
    gone, twice, other = dw.clone(), dw.clone(), dw.clone()
    gone[piece:2 * piece] = 0
    twice[:piece] *= 2
    other[2 * piece:] = dw[piece:2 * piece]
    for wrong in (gone, twice, other):
        assert bad(dh, wrong)[1] > 0.3  # (of a third of the entries nearly all)
    dh2, dw2 = grads(dloss.roll(1))
    assert min(bad(dh2, dw2)) > 0.5
    # The last rows missing from dW; the last piece missing from dh.
    short = dw - (grads(torch.where(torch.arange(T) >= T - 64, dloss, 0.0) + 1e-30)[1])
    assert bad(dh, short)[1] > 0.05
    assert bad((dh.double() - dh.double() * 0.05).to(dh.dtype), dw)[0] > 0.5


@pytest.mark.gpu
def test_no_rows_of_many_weights(cuda):
    """2^32 weights: as many threads as one launch cannot hold."""
    torch = cuda
    from jax_mlx_amd import native as nat

    w = torch.empty(1 << 18, 1 << 14, device="cuda", dtype=torch.bfloat16)
    z, t = torch.empty(0, device="cuda"), torch.empty(0, device="cuda", dtype=torch.int64)
    dw = torch.ones_like(w)
    nat.linear_xent_bwd(w[:0], w, t, z, z, need_dh=False, dw=dw)
    assert not dw.any()


@pytest.mark.gpu
def test_sums_of_more_entries_than_a_grid(cuda):
    """dh of 2^31 entries, added over pieces: the last sum's threads take
    several each.  Rows apart have the gradients of their own, so some are
    compared."""
    torch = cuda
    from jax_mlx_amd import native as nat

    T, H, V = (1 << 19) + 3, 4096, 700
    g = torch.Generator("cuda").manual_seed(8)
    w = (torch.randn(V, H, device="cuda", generator=g) * H ** -0.5).to(torch.bfloat16)
    h = torch.empty(T, H, device="cuda", dtype=torch.bfloat16)
    for a in range(0, T, 1 << 16):
        h[a:a + (1 << 16)] = torch.randn(min(1 << 16, T - a), H, device="cuda", generator=g)
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    dloss = torch.rand(T, device="cuda", generator=g)
    assert T * 256 * 2 <= 512 << 20 < T * V * 2
    _, lse = nat.linear_xent(h, w, t)
    dh = torch.full_like(h, float("nan"))
    nat.linear_xent_bwd(h, w, t, lse, dloss, need_dw=False, dh=dh)
    assert dh.isfinite().all()
    for a in (0, 70000, 262143, 400000, T - 200):
        s = slice(a, a + 200)
        ref, bound, _, _ = bounds(torch, "bf16", h[s], w, t[s], dloss[s])
        assert not out_of_bounds(torch, "bf16", dh[s], ref, bound).any(), a
