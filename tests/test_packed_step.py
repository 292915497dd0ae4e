"""The packed operators together, as a training step uses them: projection,
query / key norm with rotation, attention over packed sequences, projection,
the loss of a linear head, and back, through the package's entry points,
against torch's autograd in 64 bits on the CPU.

Tolerances, of a tensor's norm.  f32: a stage's sums of at most 512 terms are off
by under sqrt(512) 2^-24 of their norm, scores of size up to 10 turn that into
ten times as much, twelve stages there and back: 12 * 10 * 23 * 2^-24 < 2^-12.
bf16: twelve stages each round by at most 2^-8 of the norm, doubled for what the
stages behind make of it: 12 * 2 * 2^-8 < 0.1."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HQ, HKV, D, E, V = 4, 2, 64, 128, 777
LENS = [1, 70, 129, 33]
TAIL = 7  # rows in no sequence, as a fixed-size batch has
EPS = 1e-6


@pytest.fixture(scope="module")
def nat(cuda):
    from jax_mlx_amd import native

    native.load()
    return native


def inputs(torch, dtype):
    g = torch.Generator("cuda").manual_seed(21)
    T = sum(LENS) + TAIL
    mk = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)  # noqa: E731
    p = dict(x=mk(T, E), wqkv=mk(E, (HQ + 2 * HKV) * D, scale=E ** -0.5), wo=mk(HQ * D, E, scale=(HQ * D) ** -0.5),
             head=mk(V, E, scale=E ** -0.5), qw=1 + mk(D, scale=0.1), kw=1 + mk(D, scale=0.1))
    off = torch.tensor([0] + LENS, device="cuda").cumsum(0).to(torch.int32)
    pos = torch.cat([torch.arange(n) for n in LENS + [TAIL]]).to(torch.int32).cuda()
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    t[sum(LENS):] = -100
    t[5] = -100
    return p, off, pos, t


def step(torch, nat, p, off, pos, t, table):
    """(loss, gradients of every entry of p) by the package's kernels."""
    T, dtype = p["x"].shape[0], p["x"].dtype
    gemm = lambda a, b, **kw: nat.gemm(a, b, out_dtype=dtype, **kw)  # noqa: E731
    qkv = gemm(p["x"], p["wqkv"]).view(T, HQ + 2 * HKV, D)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
    norm = dict(q_weight=p["qw"], k_weight=p["kw"], eps=EPS)
    qn, kn = nat.qk_norm_rope(q, k, pos, table, **norm)
    lse = torch.zeros(HQ, T, device="cuda")
    # (Rows in no sequence are not written: they start from zeros.)
    o = nat.sdpa_packed(qn, kn, v, off, out=torch.zeros_like(qn), lse=lse)
    y = gemm(o.view(T, HQ * D), p["wo"])
    loss, zlse = nat.linear_xent(y, p["head"], t)
    w = (t >= 0).float() / (t >= 0).sum()
    dy, dhead = nat.linear_xent_bwd(y, p["head"], t, zlse, w)
    do = gemm(dy, p["wo"], trans_b=True).view(T, HQ, D)
    dwo = gemm(o.view(T, HQ * D), dy, trans_a=True)
    dqkv = torch.zeros_like(qkv)
    dqn, dkn = torch.zeros_like(qn), torch.zeros_like(kn)
    nat.sdpa_packed_bwd(qn, kn, v, do, o, lse, off, dq=dqn, dk=dkn, dv=dqkv[:, HQ + HKV:])
    _, _, dqw, dkw = nat.qk_norm_rope_bwd(q, k, dqn, dkn, pos, table, dq=dqkv[:, :HQ], dk=dqkv[:, HQ:HQ + HKV], **norm)
    dqkv = dqkv.view(T, -1)
    dx = gemm(dqkv, p["wqkv"], trans_b=True)
    dwqkv = gemm(p["x"], dqkv, trans_a=True)
    return (loss * w).sum(), dict(x=dx, wqkv=dwqkv, wo=dwo, head=dhead, qw=dqw, kw=dkw)


def reference(torch, p, off, pos, t):
    p = {n: x.double().cpu().requires_grad_() for n, x in p.items()}
    off, pos, t = off.tolist(), pos.cpu(), t.cpu()
    T = p["x"].shape[0]
    qkv = (p["x"] @ p["wqkv"]).view(T, HQ + 2 * HKV, D)
    ang = pos.double()[:, None] * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def turn(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, k, v = turn(qkv[:, :HQ], p["qw"]), turn(qkv[:, HQ:HQ + HKV], p["kw"]), qkv[:, HQ + HKV:]
    rows = []
    for a, b in zip(off, off[1:]):
        kk, vv = (x[a:b].repeat_interleave(HQ // HKV, 1).transpose(0, 1) for x in (k, v))
        z = q[a:b].transpose(0, 1) @ kk.transpose(1, 2) * D ** -0.5
        z = z.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -torch.inf)
        rows.append((torch.softmax(z, -1) @ vv).transpose(0, 1))
    o = torch.cat(rows + [torch.zeros(T - off[-1], HQ, D, dtype=torch.float64)])
    loss = torch.nn.functional.cross_entropy(o.reshape(T, HQ * D) @ p["wo"] @ p["head"].T, t, ignore_index=-100)
    loss.backward()
    return float(loss.detach()), {n: x.grad for n, x in p.items()}


@pytest.mark.parametrize("name,tol", [("f32", 2.0 ** -12), ("bf16", 0.1)])
def test_training_step(cuda, nat, name, tol):
    torch = cuda
    p, off, pos, t = inputs(torch, {"f32": torch.float32, "bf16": torch.bfloat16}[name])
    table = nat.rope_table(D)
    loss, grads = step(torch, nat, p, off, pos, t, table)
    want, refs = reference(torch, p, off, pos, t)
    assert abs(float(loss) - want) <= tol * want
    for n, ref in refs.items():
        err = float((grads[n].double().cpu() - ref).norm() / ref.norm())
        assert err <= tol, (n, err)


def test_captured_step_replays(cuda, nat):
    """One graph of the whole step, replayed on other packings and inputs with
    eager work between, against the eager step."""
    torch = cuda
    p, off, pos, t = inputs(torch, torch.bfloat16)
    table = nat.rope_table(D)
    step(torch, nat, p, off, pos, t, table)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(torch, nat, p, off, pos, t, table)  # (the GEMMs' library scratch of this stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            loss, grads = step(torch, nat, p, off, pos, t, table)
    rng = np.random.default_rng(3)
    for _ in range(3):
        cuts = np.sort(rng.integers(0, sum(LENS), len(LENS) - 1))
        off.copy_(torch.tensor([0, *cuts, sum(LENS)], dtype=torch.int32))
        p["x"].mul_(-0.9)
        t.copy_(torch.roll(t, 3))
        graph.replay()
        torch.cuda.synchronize()
        want, refs = step(torch, nat, p, off, pos, t, table)
        assert torch.equal(loss, want)
        for n, ref in refs.items():
            assert torch.equal(grads[n], ref), n
