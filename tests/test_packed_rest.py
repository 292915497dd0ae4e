"""Rows in no sequence of a packed batch (before the first, behind the last):
zeros in the outputs that the package makes, so that what goes over every row
next (projections, the head's loss, the norm weights' sums) takes in nothing
that was never written; as they were in outputs that the caller gives."""
import contextlib
import ctypes

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat(cuda):
    from jax_mlx_amd import native

    native.load()
    return native


@contextlib.contextmanager
def memory_of_nan(torch):
    """Tensors that torch allocates start as NaN."""
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True, warn_only=True)
    assert torch.utils.deterministic.fill_uninitialized_memory
    try:
        assert torch.empty(64, device="cuda").isnan().all()
        yield
    finally:
        torch.use_deterministic_algorithms(was)


def dt(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


# Every kernel: 16-bit matrix cores with and without shares, padded copies, f32
# by keys and by rows, and a wavefront a row; with few and many sequences.
CASES = [("bf16", 4, 2, 128, [9, 130, 0, 61]), ("f16", 8, 1, 64, [1411]), ("bf16", 6, 2, 96, [70, 300]),
         ("f16", 3, 1, 32, [33]), ("f32", 4, 2, 64, [9, 130]), ("f32", 8, 8, 128, [128] * 60), ("f32", 2, 1, 256, [40, 70]),
         ("bf16", 2, 1, 80, [9, 130]), ("f32", 2, 2, 48, [30]), ("bf16", 2, 1, 256, [65]), ("bf16", 2, 1, 64, [1] * 700),
         ("f32", 2, 1, 64, [1] * 700), ("bf16", 8, 8, 64, [2]), ("bf16", 2, 1, 128, [2111, 200])]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}on{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
def test_rows_in_no_sequence(cuda, nat, case, causal):
    torch = cuda
    name, Hq, Hkv, D, lens = case
    head, tail = 37, 203
    T, n = head + sum(lens) + tail, sum(lens)
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v, do = (torch.randn(T, h, D, device="cuda", generator=g).to(dt(torch, name)) for h in (Hq, Hkv, Hkv, Hq))
    off = (torch.tensor([0] + lens).cumsum(0) + head).to(torch.int32).cuda()
    lse = torch.zeros(Hq, T, device="cuda")
    inside = slice(head, head + n)

    def rest(t):
        return torch.cat([t[:head], t[head + n:]])

    with memory_of_nan(torch):
        out = nat.sdpa_packed(q, k, v, off, causal=causal, lse=lse)
        grads = nat.sdpa_packed_bwd(q, k, v, do, out, lse, off, causal=causal)
    given = [torch.full_like(t, 3.0) for t in (q, q, k, v)]
    nat.sdpa_packed(q, k, v, off, causal=causal, lse=lse, out=given[0])
    nat.sdpa_packed_bwd(q, k, v, do, given[0], lse, off, causal=causal, dq=given[1], dk=given[2], dv=given[3])
    for made, mine in zip((out, *grads), given):
        assert (rest(made) == 0).all()
        assert (rest(mine) == 3).all()
        assert torch.equal(made[inside], mine[inside]) and made[inside].isfinite().all()
    # Some made, some given.
    mine = torch.full_like(k, 3.0)
    with memory_of_nan(torch):
        dq, _, dv = nat.sdpa_packed_bwd(q, k, v, do, out, lse, off, causal=causal, dk=mine)
    assert (rest(dq) == 0).all() and (rest(mine) == 3).all() and (rest(dv) == 0).all()
    assert all(torch.equal(a[inside], b[inside]) for a, b in zip((dq, mine, dv), grads))


@pytest.mark.parametrize("name,D", [("bf16", 64), ("bf16", 80), ("f32", 64)])
def test_no_sequences(cuda, nat, name, D):
    torch = cuda
    q, k = (torch.randn(90, h, D, device="cuda").to(dt(torch, name)) for h in (4, 2))
    lse = torch.zeros(4, 90, device="cuda")
    for off in ([5], [40, 40], [0, 0, 0], [90, 90]):
        off = torch.tensor(off, dtype=torch.int32, device="cuda")
        with memory_of_nan(torch):
            out = nat.sdpa_packed(q, k, k, off, lse=lse)
            grads = nat.sdpa_packed_bwd(q, k, k, q, out, lse, off)
        assert all((t == 0).all() for t in (out, *grads))
        assert (nat.sdpa_packed(q, k, k, off, lse=lse, out=torch.full_like(q, 3.0)) == 3).all()
    assert nat.sdpa_packed(q[:0], k[:0], k[:0], off).shape == (0, 4, D)


def test_replays_with_fewer_rows(cuda, nat):
    """The rows that an earlier replay computed are zeros once they lie in no
    sequence."""
    torch = cuda
    q, k = (torch.randn(300, h, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    off = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")

    def step():
        lse = torch.zeros(4, 300, device="cuda")
        out = nat.sdpa_packed(q, k, k, off, lse=lse)
        return (out, *nat.sdpa_packed_bwd(q, k, k, q, out, lse, off))

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    for a, b, c in ((0, 100, 300), (20, 90, 120), (150, 150, 290), (0, 0, 300)):
        off.copy_(torch.tensor([a, b, c]))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y) and (x[:a] == 0).all() and (x[c:] == 0).all()


def test_outputs_of_the_argument_struct(cuda, nat):
    """C callers without zero_rest keep their rows; a call without sequences and
    with zero_rest wants outputs it can write."""
    torch = cuda
    q = torch.randn(20, 2, 64, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 3.0)
    off = torch.tensor([4], dtype=torch.int32, device="cuda")
    a = nat.sdpa_packed_args(q, q, q, out, off)
    lib, stream = nat.load(), torch.cuda.current_stream().cuda_stream
    assert lib.mfx_sdpa_packed(ctypes.byref(a), stream) == 0 and (out == 3).all()
    a.zero_rest = 1
    a.out = None
    assert lib.mfx_sdpa_packed(ctypes.byref(a), stream) == -1
    a.out = out.data_ptr()
    assert lib.mfx_sdpa_packed(ctypes.byref(a), stream) == 0 and (out == 0).all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_chain_with_the_outputs_it_makes(cuda, nat, name):
    """Norm and rotation, attention, projection, loss of a head and back, no
    buffer given, with tokens before the first and behind the last sequence:
    the gradients of the weights are those of the same chain over the tokens in
    sequences alone."""
    torch = cuda
    Hq, Hkv, D, V, H = 4, 2, 64, 500, 128
    lens, head, tail = [40, 1, 90], 11, 29
    n = sum(lens)
    T = head + n + tail
    g = torch.Generator("cuda").manual_seed(5)
    mk = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dt(torch, name))  # noqa: E731
    q, k, v = mk(T, Hq, D), mk(T, Hkv, D), mk(T, Hkv, D)
    qw, kw, wo, w = 1 + mk(D, scale=0.1), 1 + mk(D, scale=0.1), mk(Hq * D, H, scale=(Hq * D) ** -0.5), mk(V, H, scale=H ** -0.5)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    t[:head] = t[head + n:] = -100
    table = nat.rope_table(D)
    off = (torch.tensor([0] + lens).cumsum(0) + head).to(torch.int32).cuda()

    def chain(rows, off):
        q1, k1, v1, p1, t1 = (x[rows] for x in (q, k, v, pos, t))
        qn, kn = nat.qk_norm_rope(q1, k1, p1, table, q_weight=qw, k_weight=kw)
        lse = torch.zeros(Hq, q1.shape[0], device="cuda")
        o = nat.sdpa_packed(qn, kn, v1, off, lse=lse)
        y = nat.gemm(o.view(-1, Hq * D), wo, out_dtype=o.dtype)
        loss, row_lse = nat.linear_xent(y, w, t1)
        dy, dw = nat.linear_xent_bwd(y, w, t1, row_lse, torch.full_like(loss, 1.0 / n), dw_dtype=torch.float32)
        do = nat.gemm(dy, wo, trans_b=True, out_dtype=o.dtype).view(-1, Hq, D)
        dwo = nat.gemm(o.view(-1, Hq * D), dy, trans_a=True, out_dtype=torch.float32)
        dq, dk, dv = nat.sdpa_packed_bwd(qn, kn, v1, do, o, lse, off)
        dq, dk, dqw, dkw = nat.qk_norm_rope_bwd(q1, k1, dq, dk, p1, table, q_weight=qw, k_weight=kw)
        return loss, dict(dw=dw, dwo=dwo, dqw=dqw, dkw=dkw), (dq, dk, dv)

    with memory_of_nan(torch):
        loss, weights, rows = chain(slice(None), off)
        want, ref, inner = chain(slice(head, head + n), off - head)
    assert torch.equal(loss[head:head + n], want)
    for a, b in zip(rows, inner):
        assert torch.equal(a[head:head + n], b) and (a[:head] == 0).all() and (a[head + n:] == 0).all()
    # The same terms and zeros between them: sums of up to n + 40 fp32 terms in
    # another order, of which no partial sum passes the sum of magnitudes, below
    # sqrt(n) 2^3 of the result's norm; then each result's own rounding.
    for what in ref:
        a, b = weights[what].double(), ref[what].double()
        eps = torch.finfo(weights[what].dtype).eps
        tol = (n + 40) * 2.0 ** -24 * n ** 0.5 * 8 + eps
        assert a.isfinite().all() and float((a - b).norm() / b.norm()) <= tol, what
