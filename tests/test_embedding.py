"""Embedding lookup and its table's gradient (mfx_embedding,
mfx_embedding_bwd) against the formulas in 64 bits, and their refusals.

Tolerances.  A looked-up element is one fp32 product, rounded once to its type:
eps(dtype)/2 + 2^-24 of it.  A gradient's element adds n terms in fp32, at most n
deep, times the scale, plus what was there: (n + 3) half steps of the sum of
their magnitudes, and its own rounding."""
import ctypes

import numpy as np
import pytest

HALF = 2.0 ** -24
EPS = {"f32": 2.0 ** -23, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}
INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -4


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def host(t):
    return t.double().cpu().numpy()


def near(got, ref, mag, name, steps):
    assert (abs(host(got) - ref) <= EPS[name] / 2 * abs(ref) + steps * HALF * mag + TINY[name]).all()


def gradient(ids, dout, V, scale, before=None):
    """(dw, its terms' magnitude, tokens of each row) in 64 bits."""
    keep = (ids >= 0) & (ids < V)
    dw, mag = np.zeros((V, dout.shape[-1])), np.zeros((V, dout.shape[-1]))
    np.add.at(dw, ids[keep], scale * dout[keep])
    np.add.at(mag, ids[keep], abs(scale * dout[keep]))
    if before is not None:
        dw, mag = dw + before, mag + abs(before)
    return dw, mag, np.bincount(ids[keep], minlength=V)[:, None]


CASES = [
    # T, H, V, table, activations, id type, scale
    (64, 512, 1000, "bf16", "bf16", "i64", 22.6),
    (300, 4096, 777, "bf16", "bf16", "i64", 64.0),
    (257, 512, 1000, "f32", "f32", "i64", 1.0),
    (1000, 96, 5, "f16", "f16", "i32", 0.5),      # few rows: every run is long
    (4099, 130, 2000, "f32", "bf16", "i64", 1.0),  # types apart; a row's end inside a chunk
    (130, 33, 50, "bf16", "f32", "i32", -3.0),     # odd rows: no alignment
    (129, 7, 3, "f16", "f32", "i64", 1.0),
    (1, 2049, 1, "f32", "f32", "i64", 2.0),
    (65, 1, 70, "bf16", "bf16", "i64", 1.0),
    (512, 24, 40000, "bf16", "bf16", "i32", 1.0),  # the most tokens of the gradient's one launch
    (513, 33, 50, "bf16", "f32", "i32", -3.0),
    (600, 7, 3, "f16", "f32", "i64", 1.0),
    (64, 1024, 2000, "bf16", "f32", "i64", 1.0),   # a table too large for it
    (500, 8200, 2, "f32", "f32", "i64", 1.0),      # and few rows, their columns split
    (2500, 640, 1100, "f16", "f16", "i64", 1.0),   # more rows than a workgroup of the index takes at V / CUs
]
IDS = [f"T{c[0]}-H{c[1]}-V{c[2]}-{c[3]}-{c[4]}" for c in CASES]


def make(torch, case, seed=0):
    T, H, V, wname, aname, iname, scale = case
    rng = np.random.default_rng(seed)
    ids = (V * rng.random(T) ** 3).astype(np.int64).clip(max=V - 1)
    ids[rng.random(T) < 0.1] = 0
    ids[rng.random(T) < 0.05] = -100
    ids[rng.random(T) < 0.03] = V
    if T > 2:
        ids[1] = 2 ** 31 - 1 if iname == "i32" else 2 ** 40 + 3
    w = torch.from_numpy(rng.standard_normal((V, H))).to(dt(torch, wname)).cuda()
    dout = torch.from_numpy(rng.standard_normal((T, H))).to(dt(torch, aname)).cuda()
    pd = torch.from_numpy(ids).to(torch.int32 if iname == "i32" else torch.int64).cuda()
    return ids, pd, w, dout


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_lookup_and_gradient(cuda, nat, case):
    torch = cuda
    T, H, V, wname, aname, _, scale = case
    ids, pd, w, dout = make(torch, case)
    out = nat.embedding(pd, w, scale=scale, out_dtype=dt(torch, aname))
    ok = (ids >= 0) & (ids < V)
    ref = np.where(ok[:, None], host(w)[np.where(ok, ids, 0)] * np.float64(np.float32(scale)), 0.0)
    near(out, ref, abs(ref), aname, 1)
    f = np.float64(np.float32(scale))
    for name in {wname, "f32"}:
        dw = nat.embedding_bwd(pd, dout, V, scale=scale, dw_dtype=dt(torch, name))
        want, mag, n = gradient(ids, host(dout), V, f)
        near(dw, want, mag, name, n + 3)
    before = torch.from_numpy(np.random.default_rng(9).standard_normal((V, H))).to(dt(torch, wname)).cuda()
    want, mag, n = gradient(ids, host(dout), V, f, host(before))
    got = before.clone()
    assert nat.embedding_bwd(pd, dout, scale=scale, dw=got, accumulate=True) is got
    near(got, want, mag, wname, n + 3)
    none = torch.from_numpy(n[:, 0] == 0).cuda()
    assert torch.equal(got[none], before[none])  # rows without tokens, bit for bit


RUNS = [[1], [32], [33], [32, 32], [31, 34, 1], [1, 32, 33], [64], [65], [64, 64], [63, 66, 1], [1, 64, 65], [200],
        [129, 0, 3, 128], [5] * 30 + [500], [0, 0, 64, 0], [0, 32, 0, 33, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["sorted", "mixed"])
@pytest.mark.parametrize("rest", [1, 2100], ids=["small", "large"])
@pytest.mark.parametrize("runs", RUNS, ids=str)
def test_runs_about_a_pieces_length(cuda, nat, runs, rest, order):
    """Rows of 0, 1, 32, 33 .. tokens that start anywhere in a piece, against exact sums of small integers,
    in a small table (one launch) and one of more than 4 MB."""
    torch = cuda
    V, H = len(runs) + rest, 520
    ids = np.repeat(np.arange(len(runs)), runs)
    if order == "mixed":
        np.random.default_rng(1).shuffle(ids)
    dout = np.random.default_rng(2).integers(-8, 9, (len(ids), H))
    got = nat.embedding_bwd(torch.from_numpy(ids).cuda(), torch.from_numpy(dout).float().cuda(), V)
    want = np.zeros((V, H))
    np.add.at(want, ids, dout)
    assert np.array_equal(host(got), want)


@pytest.mark.gpu
def test_every_token_the_same(cuda, nat):
    torch = cuda
    T, H, V = 10000, 264, 40000
    dout = torch.randint(-8, 9, (T, H), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    ids = torch.full((T,), V - 1, device="cuda")
    got = nat.embedding_bwd(ids, dout, V, dw_dtype=torch.float32)
    assert torch.equal(got[V - 1], dout.float().sum(0)) and not got[:V - 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [90, 4000])
def test_strided_rows_and_what_lies_between(cuda, nat, V):
    """Rows of wider tensors at any alignment: the columns between stay."""
    torch = cuda
    rng = np.random.default_rng(3)
    T, H = 200, 515
    wide = torch.from_numpy(rng.standard_normal((V, H + 9))).to(torch.bfloat16).cuda()
    w = wide[:, 3:3 + H]
    ids = torch.from_numpy(rng.integers(0, V, (4, T // 4))).cuda()
    room = torch.full((4, T // 4, H + 6), 7.0, device="cuda", dtype=torch.bfloat16)
    nat.embedding(ids, w, out=room[..., 1:1 + H])
    assert torch.equal(room[..., 1:1 + H], w[ids]) and (room[..., 0] == 7).all() and (room[..., 1 + H:] == 7).all()
    dwide = torch.full((V, H + 5), 7.0, device="cuda")
    dout = torch.from_numpy(rng.integers(-8, 9, (4, T // 4, H + 2))).to(torch.float16).cuda()[..., 1:1 + H]
    nat.embedding_bwd(ids, dout, dw=dwide[:, 2:2 + H])
    want = torch.zeros(V, H, device="cuda").index_add_(0, ids.flatten(), dout.float().reshape(T, H))
    assert torch.equal(dwide[:, 2:2 + H], want) and (dwide[:, :2] == 7).all() and (dwide[:, 2 + H:] == 7).all()
    # One gradient row for every token (a sum's backward): a row stride of 0.
    one = dout[0, 0].float().clone()
    got = nat.embedding_bwd(ids.flatten(), one.expand(T, H), V)
    assert torch.equal(got, torch.bincount(ids.flatten(), minlength=V).float()[:, None] * one)


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tokens", [64, 512])
@pytest.mark.parametrize("V,H,name", [(262144, 4, "f32"), (262144, 8, "bf16"), (300001, 6, "f16"), (261632, 3, "bf16"),
                                      (2097152, 1, "f16"), (32768, 32, "f32")])
def test_one_launch_over_the_longest_tables(cuda, nat, V, H, name, tokens, accumulate):
    """Tables of narrow rows of up to 4 MB: a workgroup's rows are as many as its threads.  Tokens in the rows
    about the workgroups' ends and the table's, a run of them longer than a piece; exact sums of small integers."""
    torch = cuda
    rng = np.random.default_rng(4)
    edges = [r + d for r in (0, 512, 1024, 131072, V // 512 * 512, V) for d in (-2, -1, 0, 1)]
    edges = np.array([r for r in edges if 0 <= r < V])
    ids = rng.choice(edges, tokens)
    ids[:40] = V - 1
    ids[40:44] = 511
    ids[44:46] = -1, V
    dout = rng.integers(-1, 2, (tokens, H))
    dw = torch.full((V, H), 3.0, device="cuda", dtype=dt(torch, name))
    nat.embedding_bwd(torch.from_numpy(ids).cuda(), torch.from_numpy(dout).to(dw.dtype).cuda(), dw=dw,
                      accumulate=accumulate)
    want = np.full((V, H), 3.0 if accumulate else 0.0)
    keep = (ids >= 0) & (ids < V)
    np.add.at(want, ids[keep], dout[keep])
    assert abs(want).max() <= 256  # exact in every type
    assert np.array_equal(host(dw), want)


@pytest.mark.gpu
def test_no_tokens(cuda, nat):
    torch = cuda
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    w = torch.ones(10, 24, device="cuda")
    assert nat.embedding(ids, w).shape == (0, 24)
    dout = torch.empty(0, 24, device="cuda")
    assert not nat.embedding_bwd(ids, dout, dw=w.clone()).any()
    assert (nat.embedding_bwd(ids, dout, dw=w, accumulate=True) == 1).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda, nat):
    """A table of 5.6 GB: rows whose elements and bytes lie past 2^31 and 2^32."""
    torch = cuda
    V, H = 70000, 40000
    w = torch.empty(V, H, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 53687, 53688, 69999], device="cuda")
    vals = torch.randn(4, H, device="cuda").to(torch.bfloat16)
    w[rows] = vals
    assert torch.equal(nat.embedding(rows, w), vals)
    w.fill_(3.0)
    nat.embedding_bwd(rows, vals, dw=w)
    assert torch.equal(w[rows], vals)
    rest = torch.ones(V, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert int(w.ne(0).any(1)[rest].sum()) == 0


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda, nat):
    """A graph replayed on other tokens, with eager work between, and two streams at once."""
    torch = cuda
    T, H, V = 700, 256, 300
    g = torch.Generator("cuda").manual_seed(5)
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    dout, w = (torch.randn(n, H, device="cuda", generator=g).to(torch.bfloat16) for n in (T, V))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        nat.embedding_bwd(ids, dout, V)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = nat.embedding(ids, w, scale=3.0)
            dw = nat.embedding_bwd(ids, dout, V, scale=3.0)
    for k in range(4):
        ids.copy_(torch.randint(-1, V if k % 2 else 3, (T,), device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nat.embedding(ids, w, scale=3.0))
        assert torch.equal(dw, nat.embedding_bwd(ids, dout, V, scale=3.0))
    other = torch.randint(0, 5, (T,), device="cuda", generator=g)
    want = [nat.embedding_bwd(i, dout, V) for i in (ids, other)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, i in enumerate((ids, other)):
            with torch.cuda.stream(streams[k]):
                got[k].append(nat.embedding_bwd(i, dout, V))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[k]) for k in range(2) for x in got[k])


def test_refusals(nat):
    lib = nat.load()

    def fwd(**kw):
        a = nat.EmbeddingArgs()
        a.w, a.ids, a.out = 0x100000, 0x200000, 0x300000
        a.T, a.H, a.V, a.w_stride, a.out_stride = 8, 64, 100, 64, 64
        a.scale, a.dtype, a.out_dtype, a.ids_dtype = 1.0, nat.MFX_BF16, nat.MFX_BF16, nat.MFX_I64
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mfx_embedding(ctypes.byref(a), None)

    def bwd(**kw):
        a = nat.EmbeddingBwdArgs()
        a.dout, a.ids, a.dw = 0x100000, 0x200000, 0x300000
        a.T, a.H, a.V, a.dout_stride, a.dw_stride = 8, 64, 100, 64, 64
        a.scale, a.dtype, a.dw_dtype, a.ids_dtype = 1.0, nat.MFX_BF16, nat.MFX_BF16, nat.MFX_I64
        for k, v in kw.items():
            setattr(a, k, v)
        assert lib.mfx_embedding_bwd_workspace_size(ctypes.byref(a)) == 0 or "workspace" in kw
        return lib.mfx_embedding_bwd(ctypes.byref(a), None)

    for call, src, dst in ((fwd, "w", "out"), (bwd, "dout", "dw")):
        for bad in (dict(T=-1), dict(H=0), dict(V=0), {src: 0}, {dst: 0}, dict(ids=0), {src: 0x100001}, dict(ids=0x200004),
                    {dst + "_stride": 63}, {src + "_stride": -64}, dict(scale=float("nan")), dict(scale=float("inf"))):
            assert call(**bad) == INVALID, bad
        for bad in (dict(dtype=3), dict(ids_dtype=0), {("out_dtype" if call is fwd else "dw_dtype"): 7}, dict(T=2 ** 31),
                    dict(V=2 ** 31), dict(H=2 ** 31, w_stride=2 ** 31, out_stride=2 ** 31, dout_stride=2 ** 31, dw_stride=2 ** 31)):
            assert call(**bad) == UNSUPPORTED, bad
    assert fwd(T=2 ** 27, H=4096, w_stride=4096, out_stride=4096) == UNSUPPORTED and b"too large" in lib.mfx_last_error()
    assert bwd(V=2 ** 27, H=4096, dout_stride=4096, dw_stride=4096) == UNSUPPORTED and b"too large" in lib.mfx_last_error()
    assert bwd(T=3000, workspace=0x400000, workspace_bytes=16) == WORKSPACE
    assert bwd(T=3000, workspace=0x400010, workspace_bytes=1 << 20) == INVALID
    assert fwd(T=0, w=0, ids=0, out=0) == 0


def test_python_checks(nat):
    torch = pytest.importorskip("torch")
    w, ids = torch.zeros(10, 16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError):
        nat.embedding(ids.float(), w)
    with pytest.raises(ValueError):
        nat.embedding(torch.zeros(4, 2, dtype=torch.int64)[:, 0], w)
    with pytest.raises(ValueError):
        nat.embedding(ids, w.t())
    with pytest.raises(ValueError):
        nat.embedding(ids, w, out=torch.zeros(4, 15))
    with pytest.raises(ValueError):
        nat.embedding(ids, w)  # not on a GPU
    with pytest.raises(ValueError):
        nat.embedding_bwd(ids, torch.zeros(3, 16), 10)
    with pytest.raises(ValueError):
        nat.embedding_bwd(ids, torch.zeros(4, 16))
    with pytest.raises(ValueError):
        nat.embedding_bwd(ids, torch.zeros(4, 16), 10, accumulate=True)
    with pytest.raises(ValueError):
        nat.embedding_bwd(ids, torch.zeros(4, 16), 11, dw=w)
