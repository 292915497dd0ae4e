"""A training step from token ids to new weights, through the package's entry
points: embeddings, norms around the blocks, attention over packed sequences, the
loss of a head tied to the table, back to the table, and orthogonalised updates.
Gradients against torch's autograd in 64 bits on the CPU, the update against its
definition in 64 bits on the same gradients.

Tolerances, of a tensor's norm.  f32: a stage's sums of at most 512 terms are off
by under sqrt(512) 2^-24 of their norm, scores of size up to 10 turn that into
ten times as much, twenty stages there and back: 20 * 10 * 23 * 2^-24 < 2^-11.
bf16: twenty stages each round by at most 2^-8 of the norm, doubled for what the
stages behind make of it: 20 * 2 * 2^-8 < 0.16.  An update's products are in two
terms (f32 weights) or end in bf16 weights, and the sides are short: within 2^-13 of
the update's norm, and the weights' and the momentum's own rounding."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HQ, HKV, D, E, V, SEGMENTS = 4, 2, 64, 128, 777, 3
LENS = [1, 70, 129, 33]
TAIL = 7  # rows in no sequence, as a fixed-size batch has
EPS = 1e-6
MATRICES = ("wqkv", "wo", "mlp")
UPDATE = dict(lr=0.02, mu=0.9, weight_decay=0.1, scale=0.5)
QUINTIC = (3.4445, -4.7750, 2.0315)
AROUND = dict(post_eps=EPS, pre_eps=EPS, alpha=0.9, beta=1.1, weight_offset=1.0)
LAST = dict(pre_eps=EPS, weight_offset=1.0)


@pytest.fixture(scope="module")
def nat(cuda):
    from jax_mlx_amd import native

    native.load()
    return native


def inputs(torch, dtype):
    g = torch.Generator("cuda").manual_seed(22)
    T, S = sum(LENS) + TAIL, len(LENS)
    mk = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)  # noqa: E731
    p = dict(table=mk(V, E, scale=E ** -0.5), segments=mk(SEGMENTS, E), first=mk(E, scale=0.1),
             wqkv=mk(E, (HQ + 2 * HKV) * D, scale=E ** -0.5), qw=1 + mk(D, scale=0.1), kw=1 + mk(D, scale=0.1),
             wo=mk(HQ * D, E, scale=(HQ * D) ** -0.5), gate=1 + mk(S, E, scale=0.3), post=mk(E, scale=0.1),
             pre=mk(E, scale=0.1), mlp=mk(E, E, scale=E ** -0.5), scales=1 + mk(E, scale=0.3), last=mk(E, scale=0.1))
    off = torch.tensor([0] + LENS, device="cuda").cumsum(0).to(torch.int32)
    pos = torch.cat([torch.arange(n) for n in LENS + [TAIL]]).to(torch.int32).cuda()
    ids, t = (torch.randint(0, V, (T,), device="cuda", generator=g) for _ in range(2))
    ids[50:110] = 3  # a token of many places
    seg = torch.randint(0, SEGMENTS, (T,), device="cuda", generator=g).to(torch.int32)
    t[sum(LENS):] = -100
    return p, off, pos, ids, seg, t


def gradients(torch, nat, p, off, pos, ids, seg, t, rope):
    """(loss, gradients of every entry of p) by the package's kernels."""
    T, dtype = ids.shape[0], p["table"].dtype
    gemm = lambda a, b, **kw: nat.gemm(a, b, out_dtype=dtype, **kw)  # noqa: E731
    x, s = nat.embedding(ids, p["table"], scale=E ** 0.5), nat.embedding(seg, p["segments"])
    first = dict(pre_weight=p["first"], **LAST)
    r0, h0 = nat.residual_norm(x, s, **first)
    qkv = gemm(h0, p["wqkv"]).view(T, HQ + 2 * HKV, D)
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]
    norm = dict(q_weight=p["qw"], k_weight=p["kw"], eps=EPS)
    qn, kn = nat.qk_norm_rope(q, k, pos, rope, **norm)
    lse = torch.zeros(HQ, T, device="cuda")
    o = nat.sdpa_packed(qn, kn, v, off, out=torch.zeros_like(qn), lse=lse)
    y1 = gemm(o.view(T, HQ * D), p["wo"])
    around = dict(gate=p["gate"], seq_offsets=off, post_weight=p["post"], pre_weight=p["pre"], **AROUND)
    r1, h1 = nat.residual_norm(r0, y1, **around)
    y2 = gemm(h1, p["mlp"])
    last = dict(gate=p["scales"], pre_weight=p["last"], **LAST)
    _, h2 = nat.residual_norm(r1, y2, **last)
    loss, zlse = nat.linear_xent(h2, p["table"], t)
    w = (t >= 0).float() / (t >= 0).sum()

    dh2, dtable = nat.linear_xent_bwd(h2, p["table"], t, zlse, w)
    dr1, dy2, dscales, _, dlast = nat.residual_norm_bwd(r1, y2, None, dh2, dy=dh2, **last)
    dh1, dmlp = gemm(dy2, p["mlp"], trans_b=True), gemm(h1, dy2, trans_a=True)
    dr0, dy1, dgate, dpost, dpre = nat.residual_norm_bwd(r0, y1, dr1, dh1, dx=dr1, dy=dh1, **around)
    do = gemm(dy1, p["wo"], trans_b=True).view(T, HQ, D)
    dwo = gemm(o.view(T, HQ * D), dy1, trans_a=True)
    dqkv = torch.zeros_like(qkv)
    dqn, dkn = torch.zeros_like(qn), torch.zeros_like(kn)
    nat.sdpa_packed_bwd(qn, kn, v, do, o, lse, off, dq=dqn, dk=dkn, dv=dqkv[:, HQ + HKV:])
    _, _, dqw, dkw = nat.qk_norm_rope_bwd(q, k, dqn, dkn, pos, rope, dq=dqkv[:, :HQ], dk=dqkv[:, HQ:HQ + HKV], **norm)
    dqkv = dqkv.view(T, -1)
    dh0, dwqkv = gemm(dqkv, p["wqkv"], trans_b=True), gemm(h0, dqkv, trans_a=True)
    dx, ds, _, _, dfirst = nat.residual_norm_bwd(x, s, dr0, dh0, **first)
    nat.embedding_bwd(ids, dx, dw=dtable, scale=E ** 0.5, accumulate=True)
    dsegments = nat.embedding_bwd(seg, ds, SEGMENTS)
    return (loss * w).sum(), dict(table=dtable, segments=dsegments, first=dfirst, wqkv=dwqkv, qw=dqw, kw=dkw, wo=dwo,
                                  gate=dgate, post=dpost, pre=dpre, mlp=dmlp, scales=dscales, last=dlast)


def step(torch, nat, p, momentum, *batch):
    loss, grads = gradients(torch, nat, p, *batch)
    for n in MATRICES:
        nat.muon_update(p[n], grads[n], momentum[n], **UPDATE)
    return loss, grads


def reference(torch, p, off, pos, ids, seg, t):
    p = {n: x.double().cpu().requires_grad_() for n, x in p.items()}
    off, pos, ids, seg, t = off.tolist(), pos.cpu(), ids.cpu(), seg.cpu().long(), t.cpu()
    T = len(ids)
    rms = lambda x, w: x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w)  # noqa: E731
    ang = pos.double()[:, None] * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def turn(x, w):
        x = rms(x, w - 1)
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    r0 = E ** 0.5 * p["table"][ids] + p["segments"][seg]
    qkv = (rms(r0, p["first"]) @ p["wqkv"]).view(T, HQ + 2 * HKV, D)
    q, k, v = turn(qkv[:, :HQ], p["qw"]), turn(qkv[:, HQ:HQ + HKV], p["kw"]), qkv[:, HQ + HKV:]
    rows = []
    for a, b in zip(off, off[1:]):
        kk, vv = (x[a:b].repeat_interleave(HQ // HKV, 1).transpose(0, 1) for x in (k, v))
        z = q[a:b].transpose(0, 1) @ kk.transpose(1, 2) * D ** -0.5
        z = z.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -torch.inf)
        rows.append((torch.softmax(z, -1) @ vv).transpose(0, 1))
    rest = T - off[-1]
    o = torch.cat(rows + [torch.zeros(rest, HQ, D, dtype=torch.float64)])
    y1 = o.reshape(T, HQ * D) @ p["wo"]
    gate = torch.cat([p["gate"].repeat_interleave(torch.tensor(off).diff(), 0), torch.zeros(rest, E, dtype=torch.float64)])
    r1 = AROUND["alpha"] * r0 + AROUND["beta"] * gate * rms(y1, p["post"])
    r2 = r1 + p["scales"] * (rms(r1, p["pre"]) @ p["mlp"])
    loss = torch.nn.functional.cross_entropy(rms(r2, p["last"]) @ p["table"].T, t, ignore_index=-100)
    loss.backward()
    return float(loss.detach()), {n: x.grad for n, x in p.items()}


def updated(torch, w, g, momentum):
    """(w, momentum, the update's norm) by the definition in 64 bits."""
    w, g, b = (x.double().cpu() for x in (w, g, momentum))
    mu, lr = (float(np.float32(UPDATE[n])) for n in ("mu", "lr"))
    b = mu * b + (1 - mu) * g
    u = mu * b + (1 - mu) * g
    x = u / u.norm()
    wide = x.shape[0] <= x.shape[1]
    for _ in range(5):
        a2, a4, a6 = (float(np.float32(v)) for v in QUINTIC)
        s = x @ x.T if wide else x.T @ x
        f = a2 * torch.eye(len(s), dtype=s.dtype) + a4 * s + a6 * s @ s
        x = f @ x if wide else x @ f
    x = lr * UPDATE["scale"] * x
    return (1 - lr * float(np.float32(UPDATE["weight_decay"]))) * w - x, b, float(x.norm())


@pytest.mark.parametrize("name,tol", [("f32", 2.0 ** -11), ("bf16", 0.16)])
def test_step(cuda, nat, name, tol):
    torch = cuda
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[name]
    p, *batch = inputs(torch, dtype)
    momentum = {n: 0.001 * torch.randn_like(p[n]) for n in MATRICES}
    before = {n: (p[n].clone(), momentum[n].clone()) for n in MATRICES}
    want, refs = reference(torch, p, *batch)
    loss, grads = step(torch, nat, p, momentum, *batch, nat.rope_table(D))
    assert abs(float(loss) - want) <= tol * want
    for n, ref in refs.items():
        err = float((grads[n].double().cpu() - ref).norm() / ref.norm())
        assert err <= tol, (n, err)
    half = torch.finfo(dtype).eps / 2
    for n, (w, b) in before.items():
        w, b, size = updated(torch, w, grads[n], b)
        assert float((p[n].double().cpu() - w).norm()) <= 2.0 ** -13 * size + 2 * half * float(w.norm())
        assert float((momentum[n].double().cpu() - b).norm()) <= 2 * half * float(b.norm())


def test_captured_step_replays(cuda, nat):
    """One graph of the step, weights and momentum updated in place, replayed on
    other packings and tokens with eager work between, against the eager step."""
    torch = cuda
    p, *batch = inputs(torch, torch.bfloat16)
    off, pos, ids, seg, t = batch
    rope = nat.rope_table(D)
    momentum = {n: torch.zeros_like(p[n], dtype=torch.float32) for n in MATRICES}
    copy = lambda d: {n: x.clone() for n, x in d.items()}  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(torch, nat, copy(p), copy(momentum), *batch, rope)  # (the GEMMs' library scratch of this stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss, grads = step(torch, nat, p, momentum, *batch, rope)
    rng = np.random.default_rng(4)
    for _ in range(3):
        cuts = np.sort(rng.integers(0, sum(LENS), len(LENS) - 1))
        off.copy_(torch.tensor([0, *cuts, sum(LENS)], dtype=torch.int32))
        ids.copy_(torch.roll(ids, 5))
        t.copy_(torch.roll(t, 3))
        p2, momentum2 = copy(p), copy(momentum)
        want, refs = step(torch, nat, p2, momentum2, *batch, rope)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        for got, ref in ((grads, refs), (p, p2), (momentum, momentum2)):
            for n in ref:
                assert torch.equal(got[n], ref[n]), n
