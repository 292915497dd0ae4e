"""Attention over packed sequences (mfx_sdpa_packed, mfx_sdpa_packed_bwd)
against softmax attention of each sequence alone in 64 bits, its isolation of
sequences and its refusals.

Tolerances.  Forward, 16 bits: each probability is rounded to the type (half a
step, eps/2 relative) as the row sums take it, so the mean they form of V is off
by at most eps/2 of the mean of |V| around it, counted twice for numerator and
denominator; the output's rounding adds eps/2.  fp32's own steps (products of D
terms, exp2 of scores up to 2^6 in log2 units: 2^-17 relative) are below that
for 16 bits and are the whole of it for f32: 2^-15 of the mean of |V|.
lse: the 16-bit kernels sum the rounded probabilities, a sum off by at most
eps/2 relative, its log2 by eps/2 / ln 2; fp32 adds 2^-13.
Backward: P = exp2(s - lse) is off by that eps/2 relative, dS = P (dP - delta)
by it, by its own rounding (eps/2) and by delta's, whose output is off by
3 eps/2 of the mean of |V|: 5 eps/2 of the terms' magnitudes at most, and every
gradient is a sum of such terms.  fp32's steps add 2^-14, the output's rounding
eps/2.  (For f32 there is only the 2^-14.)"""
import ctypes

import numpy as np
import pytest

EPS = {"f32": 2.0 ** -23, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def reference(q, k, v, g, lens, causal, scale):
    """out, dq, dk, dv and the magnitude each is bounded by; lse [Hq, T].
    CPU double tensors [T, H, D]; rows behind the last sequence stay zero."""
    import torch

    G = q.shape[1] // k.shape[1]
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    mo, mq, mk, mv = (torch.zeros_like(t) for t in (q, q, k, v))
    lse = torch.zeros(q.shape[1], q.shape[0], dtype=torch.float64)
    a = 0
    for n in lens:
        b = a + n
        for h in range(q.shape[1] if n else 0):
            j = h // G
            s = q[a:b, h] @ k[a:b, j].T * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -torch.inf)
            lse[h, a:b] = torch.logsumexp(s, 1) / np.log(2)
            p = torch.softmax(s, 1)
            o[a:b, h] = p @ v[a:b, j]
            mo[a:b, h] = p @ v[a:b, j].abs()
            dp = g[a:b, h] @ v[a:b, j].T
            mdp = g[a:b, h].abs() @ v[a:b, j].abs().T
            delta = (g[a:b, h] * o[a:b, h]).sum(1, keepdim=True)
            mdelta = (g[a:b, h].abs() * mo[a:b, h]).sum(1, keepdim=True)
            ds, mds = p * (dp - delta) * scale, p * (mdp + mdelta) * abs(scale)
            dq[a:b, h] = ds @ k[a:b, j]
            mq[a:b, h] = mds @ k[a:b, j].abs()
            dk[a:b, j] += ds.T @ q[a:b, h]
            mk[a:b, j] += mds.T @ q[a:b, h].abs()
            dv[a:b, j] += p.T @ g[a:b, h]
            mv[a:b, j] += p.T @ g[a:b, h].abs()
        a = b
    return (o, dq, dk, dv), (mo, mq, mk, mv), lse


def make(torch, name, lens, Hq, Hkv, D, tail=0, seed=0, layout="thd"):
    """q, k, v, g on the GPU: tokens of all sequences and `tail` behind them."""
    gen = torch.Generator("cuda").manual_seed(seed)
    T = sum(lens) + tail

    def mk(H):
        if layout == "htd":
            return torch.randn(H, T, D, device="cuda", generator=gen).to(dt(torch, name)).transpose(0, 1)
        return torch.randn(T, H, D, device="cuda", generator=gen).to(dt(torch, name))

    off = torch.tensor([0] + list(lens), device="cuda").cumsum(0).to(torch.int32)
    return mk(Hq), mk(Hkv), mk(Hkv), mk(Hq), off


def check_all(torch, nat, name, lens, Hq, Hkv, D, causal=True, tail=0, layout="thd", scale=None, seed=0):
    q, k, v, g, off = make(torch, name, lens, Hq, Hkv, D, tail, seed, layout)
    T, n = q.shape[0], sum(lens)
    fill = lambda t: torch.full_like(t, 3.0)  # noqa: E731
    out, dq, dk, dv = fill(q), fill(q), fill(k), fill(v)
    lse = torch.full((Hq, T), 3.0, device="cuda")
    nat.sdpa_packed(q, k, v, off, causal=causal, scale=scale, out=out, lse=lse)
    nat.sdpa_packed_bwd(q, k, v, g, out, lse, off, causal=causal, scale=scale, dq=dq, dk=dk, dv=dv)
    cpu = [t.double().cpu() for t in (q, k, v, g)]
    refs, mags, rl = reference(*cpu, lens, causal, D ** -0.5 if scale is None else scale)
    e = EPS[name]
    for what, got, ref, mag in zip("out dq dk dv".split(), (out, dq, dk, dv), refs, mags):
        got = got.double().cpu()
        tol = e / 2 * ref.abs() + (2 * e / 2 + 2.0 ** -15 if what == "out" else 5 * e / 2 + 2.0 ** -14) * mag
        bad = (got[:n] - ref[:n]).abs() > tol[:n] + TINY[name]
        assert not bad.any(), (what, bad.nonzero()[:3], (got[:n] - ref[:n]).abs().max())
        assert (got[n:] == 3).all(), what
    assert ((lse[:, :n].double().cpu() - rl[:, :n]).abs() <= e / 2 / np.log(2) + 2.0 ** -13).all()
    assert (lse[:, n:] == 3).all()


LENS = [1, 37, 128, 0, 64, 5, 129, 200]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 80])
@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_mixed_lengths(cuda, nat, name, D, causal):
    check_all(cuda, nat, name, LENS, 4, 2, D, causal, tail=70)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    ("bf16", [1], 1, 1, 64), ("bf16", [1] * 200, 8, 8, 128), ("f32", [1, 2, 3], 8, 1, 64), ("bf16", [0, 0, 0], 2, 2, 64),
    ("f16", [127, 128, 129], 16, 8, 128), ("bf16", [1000], 8, 8, 64), ("bf16", [0, 700, 0, 33], 24, 8, 128),
    ("f32", [300, 1, 300], 3, 3, 256), ("f32", [513], 16, 16, 32), ("bf16", [33, 65], 5, 5, 256),
], ids=lambda c: f"{c[0]}-{len(c[1])}x{max(c[1])}-{c[2]}:{c[3]}-D{c[4]}")
def test_lengths_and_heads(cuda, nat, case):
    name, lens, Hq, Hkv, D = case
    check_all(cuda, nat, name, lens, Hq, Hkv, D, tail=3)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_head_major_and_scale(cuda, nat, name):
    check_all(cuda, nat, name, [70, 130, 1], 4, 2, 64, layout="htd", tail=60)
    check_all(cuda, nat, name, [70, 130, 1], 4, 2, 64, scale=-0.2)
    check_all(cuda, nat, name, [70, 130, 1], 4, 2, 64, scale=0.0)


@pytest.mark.gpu
def test_many_sequences(cuda, nat):
    """Both ways of finding a block: up to 512 sequences and beyond."""
    rng = np.random.default_rng(1)
    for n in (65, 512, 513, 1300):
        lens = rng.integers(0, 4, n).tolist()
        lens[n // 2] = 300
        check_all(cuda, nat, "bf16", lens, 2, 1, 64, seed=n)
        check_all(cuda, nat, "f32", lens, 2, 1, 64, seed=n)


@pytest.mark.gpu
def test_more_sequences_than_tokens(cuda, nat):
    """Empty sequences beside a few tokens, under and over 512 of them."""
    for n, at in ((400, (0, 200, 399)), (1500, (3, 700, 1499))):
        lens = [0] * n
        for i, s in enumerate(at):
            lens[s] = (1, 40, 150)[i]
        for name in ("bf16", "f32"):
            check_all(cuda, nat, name, lens, 2, 1, 64, tail=2, seed=n)


@pytest.mark.gpu
def test_longer_sequences(cuda, nat):
    check_all(cuda, nat, "bf16", [1500, 20, 700], 8, 2, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # name, lengths, heads, head size: key blocks of one share up to eight.
    ("bf16", [1411], 8, 1, 128),
    ("f16", [1000, 300, 77], 8, 1, 64),
    ("bf16", [700, 0, 129, 640], 6, 2, 96),
    ("bf16", [1300] + [40] * 70, 8, 2, 64),
    ("f16", [900, 901], 4, 4, 128),
    # and query blocks too (more than 2048 tokens, few heads).
    ("bf16", [2111, 200], 2, 1, 128),
    ("f16", [1200, 3, 1025], 2, 2, 64),
    ("bf16", [2300], 1, 1, 32),
], ids=lambda c: f"{c[0]}-{len(c[1])}-{c[2]}on{c[3]}-{c[4]}")
def test_shared_key_blocks(cuda, nat, case):
    name, lens, Hq, Hkv, D = case
    check_all(cuda, nat, name, lens, Hq, Hkv, D, tail=5)


@pytest.mark.gpu
def test_shared_key_blocks_repeat(cuda, nat):
    """Shares of a key block are counted in a workspace that may hold anything,
    by eager and captured calls, and give the same bits each time."""
    torch = cuda
    q, k, v, g, off = make(torch, "bf16", [2000, 24, 512], 8, 1, 128)
    T = q.shape[0]
    lse = torch.zeros(8, T, device="cuda")
    o = torch.empty_like(q)
    ws = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")

    def step():
        nat.sdpa_packed(q, k, v, off, out=o, lse=lse)
        return nat.sdpa_packed_bwd(q, k, v, g, o, lse, off, workspace=ws)

    ws.fill_(255)
    first = [t.clone() for t in step()]
    for fill in (0, 1, 127):
        ws.fill_(fill)
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    for lens in ([2536, 0, 0], [2000, 24, 512], [3, 2200, 333]):
        off.copy_(torch.tensor([0] + lens).cumsum(0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        ws.fill_(85)
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["thd", "htd"])
@pytest.mark.parametrize("name,D", [("bf16", 64), ("f16", 96), ("f32", 64), ("bf16", 80)])
def test_sequences_do_not_see_each_other(cuda, nat, name, D, layout):
    """Rows of other sequences, and rows in none, may hold anything."""
    torch = cuda
    lens, tail = [70, 33, 130], 40
    q, k, v, g, off = make(torch, name, lens, 4, 2, D, tail, 3, layout)
    want = [nat.sdpa_packed(q, k, v, off, lse=(lse := torch.zeros(4, q.shape[0], device="cuda")))]
    want += nat.sdpa_packed_bwd(q, k, v, g, want[0], lse, off)
    for value in (float("nan"), float("inf")):
        q2, k2, v2, g2 = (t.clone(memory_format=torch.preserve_format) for t in (q, k, v, g))
        for t in (q2, k2, v2, g2):
            t[70:103] = value
            t[233:] = value
        lse2 = torch.full((4, q.shape[0]), float("nan"), device="cuda")
        o2 = torch.full_like(q2, float("nan"))
        nat.sdpa_packed(q2, k2, v2, off, out=o2, lse=lse2)
        got = [o2, *nat.sdpa_packed_bwd(q2, k2, v2, g2, o2, lse2, off)]
        for a, b in zip(want, got):
            assert torch.equal(a[:70], b[:70]) and torch.equal(a[103:233], b[103:233])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_each_sequence_alone_gives_the_same(cuda, nat, name):
    """A sequence's rows do not depend on what it is packed with."""
    torch = cuda
    lens = [200, 5, 131]
    q, k, v, g, off = make(torch, name, lens, 4, 2, 128)
    o = nat.sdpa_packed(q, k, v, off)
    a = 0
    for n in lens:
        one = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        assert torch.equal(nat.sdpa_packed(q[a:a + n], k[a:a + n], v[a:a + n], one), o[a:a + n])
        a += n
    # Offsets that start behind the first token, with rows before it.
    shifted = nat.sdpa_packed(q, k, v, off[1:], out=torch.full_like(q, 3.0))
    assert (shifted[:200] == 3).all() and torch.equal(shifted[200:], o[200:])


@pytest.mark.gpu
def test_captured_step_replays_with_other_lengths(cuda, nat):
    torch = cuda
    q, k, v, g, off = make(torch, "bf16", [100, 50, 150], 8, 2, 128)

    def step():
        lse = torch.zeros(8, 300, device="cuda")
        o = nat.sdpa_packed(q, k, v, off, lse=lse)
        return (o, *nat.sdpa_packed_bwd(q, k, v, g, o, lse, off))

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    for lens in ([300, 0, 0], [1, 298, 1], [100, 100, 100]):
        off.copy_(torch.tensor([0] + lens).cumsum(0))
        q.mul_(1.01)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [[0, 400, 100], [-50, 20, 1000], [300, 200, 100], [0, 0, 0], [250, 250, 300]])
@pytest.mark.parametrize("name,D", [("bf16", 64), ("bf16", 96), ("f32", 64), ("f32", 48)])
def test_offsets_out_of_order_stay_inside(cuda, nat, name, D, off):
    """Only that the guard rows around the tensors are left alone."""
    torch = cuda
    big = [torch.full((500, 2, D), 5.0, device="cuda", dtype=dt(torch, name)) for _ in range(8)]
    q, k, v, g, o, dq, dk, dv = (t[100:400] for t in big)
    lse = torch.full((2, 300), 1.0, device="cuda")
    offs = torch.tensor(off, device="cuda", dtype=torch.int32)
    nat.sdpa_packed(q, k, v, offs, out=o, lse=lse)
    nat.sdpa_packed_bwd(q, k, v, g, o, lse, offs, dq=dq, dk=dk, dv=dv)
    for t in big:
        assert (t[:100] == 5).all() and (t[400:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq", [(512, 8), (2100, 2)])
def test_overlapping_offsets_stay_inside_the_workspace(cuda, nat, T, Hq):
    """200 sequences that are each the whole batch have more blocks than the
    workspace has shares for."""
    torch = cuda
    q, k, v, g, _ = make(torch, "bf16", [T], Hq, 1, 64)
    lse = torch.zeros(Hq, T, device="cuda")
    off = torch.tensor([0, T] * 200, device="cuda", dtype=torch.int32)
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    args = nat.sdpa_packed_bwd_args(q, k, v, g, out, lse, dq, dk, dv, off)
    import ctypes

    need = int(nat.load().mfx_sdpa_packed_bwd_workspace_size(ctypes.byref(args)))
    ws = torch.full((need + (1 << 26),), 7, dtype=torch.uint8, device="cuda")
    nat.sdpa_packed_bwd(q, k, v, g, out, lse, off, dq=dq, dk=dk, dv=dv, workspace=ws[:need])
    assert (ws[need:] == 7).all()


@pytest.mark.gpu
def test_gradient_against_differences(cuda, nat):
    torch = cuda
    q, k, v, g, off = make(torch, "f32", [20, 40], 2, 1, 64, seed=5)
    lse = torch.zeros(2, 60, device="cuda")
    o = nat.sdpa_packed(q, k, v, off, lse=lse)
    grads = nat.sdpa_packed_bwd(q, k, v, g, o, lse, off)

    def f(q, k, v):
        return float((nat.sdpa_packed(q, k, v, off).double() * g.double()).sum())

    h = 2.0 ** -6
    for i, d in enumerate(grads):
        step = d / d.norm()
        xs = [[t + s * h * step if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1)]
        num = (f(*xs[0]) - f(*xs[1])) / (2 * h)
        # Outputs (of size 1, 60 * 2 * 64 of them) off by 2^-15 at random over
        # 2 h, and the third derivative's h^2 / 6 of a softmax's, below h^2.
        tol = 2.0 ** -15 * (60 * 2 * 64) ** 0.5 * 2 / (2 * h) + h * h * float(d.norm())
        assert abs(num - float(d.norm())) <= tol


# ---- selection and refusals (no GPU needed) --------------------------------------

def test_kernel_selection(nat):
    import torch

    off = torch.tensor([0, 10], dtype=torch.int32)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)  # noqa: E731
    names = {(torch.bfloat16, 128): "packed_bf16_d128", (torch.float16, 32): "packed_f16_d32",
             (torch.bfloat16, 96): "packed_bf16_d96", (torch.float32, 64): "packed_f32_d64",
             (torch.float32, 80): "packed_generic", (torch.bfloat16, 72): "packed_generic"}
    for (dtype, D), name in names.items():
        q, k = z(10, 4, D, dtype=dtype), z(10, 2, D, dtype=dtype)
        assert nat.sdpa_packed_kernel_name(q, k, k, off) == name
        assert nat.sdpa_packed_bwd_kernel_name(q, k, k, off) == name
    q, k = z(10, 4, 256), z(10, 2, 256)
    assert nat.sdpa_packed_kernel_name(q, k, k, off) == "packed_generic"
    q, k = z(10, 4, 256, dtype=torch.float32), z(10, 2, 256, dtype=torch.float32)
    assert nat.sdpa_packed_kernel_name(q, k, k, off) == "packed_f32_d256"
    assert nat.sdpa_packed_bwd_kernel_name(q, k, k, off) == "packed_generic"
    # Rows off 16 bytes; no tokens; no sequences.
    q = z(10, 4, 65)[:, :, 1:]
    assert nat.sdpa_packed_kernel_name(q, q, q, off) == "packed_generic"
    q = z(10, 4, 64)
    assert nat.sdpa_packed_kernel_name(q[:0], q[:0], q[:0], off) == "none"
    assert nat.sdpa_packed_kernel_name(q, q, q, off[:1]) == "none"


def _args(nat, bwd, **over):
    a = (nat.SdpaPackedBwdArgs if bwd else nat.SdpaPackedArgs)()
    names = ("q", "k", "v", "dout", "out", "lse", "dq", "dk", "dv") if bwd else ("q", "k", "v", "out", "lse")
    for i, n in enumerate(names):
        setattr(a, n, 0x100000 * (i + 1))
    a.seq_offsets = 0x80
    a.T, a.num_seqs, a.Hq, a.Hkv, a.D = 100, 3, 4, 2, 64
    for n, _ in a._fields_:
        if n.endswith("_strides"):
            h = 2 if n[:2] in ("k_", "v_", "dk", "dv") else 4
            getattr(a, n)[:] = [64, h * 64, 1]
    a.scale, a.causal, a.dtype = 0.125, 1, nat.MFX_BF16
    for n, val in over.items():
        if isinstance(val, list):
            getattr(a, n)[:] = val
        else:
            setattr(a, n, val)
    return a


BAD = [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(seq_offsets=0), dict(T=-1), dict(num_seqs=-1), dict(Hq=0),
       dict(Hkv=0), dict(Hkv=3), dict(D=0), dict(D=257), dict(dtype=7), dict(scale=float("nan")),
       dict(scale=float("inf")), dict(T=1 << 31), dict(Hq=1 << 17, Hkv=1), dict(num_seqs=1 << 31),
       dict(q_strides=[64, 256, 2]), dict(v_strides=[64, 128, 0]), dict(o_strides=[64, 256, 3])]


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("over", BAD, ids=[",".join(o) for o in BAD])
def test_refuses(nat, bwd, over):
    lib = nat.load()
    fn = "mfx_sdpa_packed_bwd" if bwd else "mfx_sdpa_packed"
    a = _args(nat, bwd, **over)
    assert getattr(lib, fn)(ctypes.byref(a), None) in (-1, -2) and lib.mfx_last_error()
    assert getattr(lib, fn + "_kernel_name")(ctypes.byref(a)) is None


def test_refuses_null_args_and_workspace(nat):
    lib = nat.load()
    assert lib.mfx_sdpa_packed(None, None) == -1 and lib.mfx_sdpa_packed_bwd(None, None) == -1
    assert lib.mfx_sdpa_packed_bwd_workspace_size(None) == 0
    for lse in (dict(lse=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(dout=0)):
        assert lib.mfx_sdpa_packed_bwd(ctypes.byref(_args(nat, True, **lse)), None) == -1
    need = lib.mfx_sdpa_packed_bwd_workspace_size(ctypes.byref(_args(nat, True)))
    assert need >= 4 * 100 * 4
    a = _args(nat, True, workspace=0x10000000, workspace_bytes=need - 1)
    assert lib.mfx_sdpa_packed_bwd(ctypes.byref(a), None) == -4
    a = _args(nat, True, workspace=0x10000004, workspace_bytes=need)
    assert lib.mfx_sdpa_packed_bwd(ctypes.byref(a), None) == -1


def test_wrapper_refuses(nat):
    import torch

    q, k, off = torch.zeros(9, 4, 64), torch.zeros(9, 2, 64), torch.tensor([0, 9], dtype=torch.int32)
    for args, err in (((q, k, k, off), ValueError), ((q[0], k, k, off), ValueError), ((q, k[:8], k[:8], off), ValueError),
                      ((q, k, k[:, :1], off), ValueError), ((q, k.half(), k.half(), off), ValueError),
                      ((q, k, k, off.long()), TypeError), ((q, k, k, off[:0]), ValueError)):
        with pytest.raises(err):  # (the first: host tensors)
            nat.sdpa_packed(*args)
    with pytest.raises(ValueError):
        nat.sdpa_packed(q, k, k, off, lse=torch.zeros(9, 4, dtype=torch.float64))
    with pytest.raises(ValueError):
        nat.sdpa_packed(q, k, k, off, out=torch.zeros(9, 2, 64))
