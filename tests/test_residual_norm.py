"""The norms around a block with its gate and the residual sum
(mfx_residual_norm, mfx_residual_norm_bwd) against the formulas in 64 bits, and
their refusals.

Tolerances, in half steps of fp32 (2^-24) of a magnitude, beside each output's own
rounding.  A sum of squares over a row is at most 32 + 10 adds deep in a lane and
between lanes, halved by the root; with the root, a division and up to six products
and an add, r is off by under 40 half steps of m = |alpha x| + |beta g z|.  That
moves r / rms(r) by as many of e = (m + |r| p) / rms(r), p = mean(|r| m) /
mean(r^2), and h by twice as many of e w (its own steps).  The backward's terms pass
up to three times as many, 128; a sum over T rows adds T."""
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
    return None if t is None else t.double().cpu().numpy()


def near(got, ref, mag, name, steps, what=""):
    off = abs(host(got) - ref) - (EPS[name] / 2 * abs(ref) + steps * HALF * mag + TINY[name])
    assert (off <= 0).all(), (what, off.max())


def mean(v):
    return v.mean(-1, keepdims=True)


class Ref:
    """The formulas and their magnitudes in 64 bits; gate [T, H] rows (0 where a token has none)."""

    def __init__(self, x, y, gate, has, wp, wn, post_eps, pre_eps, alpha, beta, o):
        y = np.where(has[:, None], y, 0.0)
        self.wp = 1.0 if wp is None else o + wp
        self.wn = 1.0 if wn is None else o + wn
        self.iy = 1.0 if post_eps is None else 1 / np.sqrt(mean(y * y) + post_eps)
        self.yh = y * self.iy
        self.z = self.yh * self.wp
        self.g, self.alpha, self.beta, self.pre = gate, alpha, beta, pre_eps is not None
        self.post = post_eps is not None
        self.r = alpha * x + beta * gate * self.z
        self.m = abs(alpha * x) + abs(beta * gate * self.z)
        if self.pre:
            self.ir = 1 / np.sqrt(mean(self.r ** 2) + pre_eps)
            self.p = mean(abs(self.r) * self.m) / np.maximum(mean(self.r ** 2), 1e-300)
            self.rh = self.r * self.ir
            self.e = self.ir * (self.m + abs(self.r) * self.p)

    def backward(self, dr, dh):
        d, dm = dr.copy(), abs(dr)
        out = {}
        if self.pre:
            u = dh * self.wn
            d = d + self.ir * (u - self.rh * mean(u * self.rh))
            dm = dm + self.ir * (1 + self.p) * (abs(u) + 2 * self.e * mean(abs(u) * self.e))
            out["wn"] = (dh * self.rh).sum(0), (abs(dh) * self.e).sum(0)
        out["x"] = self.alpha * d, abs(self.alpha) * dm
        dz, dzm = self.beta * self.g * d, abs(self.beta * self.g) * dm
        out["gate"] = self.beta * d * self.z, abs(self.beta) * dm * abs(self.z)
        if self.post:
            v, vm = dz * self.wp, dzm * abs(self.wp)
            out["wp"] = (dz * self.yh).sum(0), (dzm * abs(self.yh)).sum(0)
            out["y"] = (self.iy * (v - self.yh * mean(v * self.yh)),
                        self.iy * (vm + 2 * abs(self.yh) * mean(vm * abs(self.yh))))
        else:
            out["y"] = dz, dzm
        return out


CASES = [
    # T, H, block, stream, params, gate, gate type, lens, post_eps, pre_eps, alpha, beta, offset
    (5, 4096, "bf16", "bf16", "bf16", None, "bf16", None, None, 1e-6, 1.0, 1.0, 0.0),
    (600, 4096, "bf16", "f32", "f32", None, "bf16", None, 1e-6, 1e-6, 1.0, 0.5, 1.0),
    (37, 1152, "f16", "f16", "f16", "seq", "f16", [9, 0, 1, 20], 1e-6, 1e-5, 1.0, 1.0, 0.0),
    (300, 512, "f32", "f32", "f32", "feature", "f32", None, None, 1e-6, 0.7, -2.0, 0.0),
    (129, 1000, "bf16", "bf16", "f32", "token", "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 1.0),
    (1000, 96, "bf16", "f32", "bf16", "seq", "f32", [1, 333, 0, 0, 64, 500, 2], 1e-6, 1e-6, 1.0, 1.0, 0.0),
    (70, 33, "f16", "f32", "f32", "feature", "f32", None, 1e-6, None, 1.0, 1.0, 0.0),   # odd rows, no h
    (3, 1, "f32", "f32", "f32", "token", "f16", None, 1e-3, 1e-3, 1.0, 1.0, 0.0),
    (1, 8191, "bf16", "bf16", "bf16", None, "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 1.0),
    (9, 16384, "f16", "f16", "f32", "feature", "f16", None, 1e-6, 1e-6, 1.0, 1.0, 0.0),
    (4, 32767, "bf16", "f32", "bf16", "seq", "bf16", [1, 2], 1e-6, 1e-6, 1.0, 1.0, 0.0),
    (2100, 2048, "bf16", "bf16", None, "feature", "bf16", None, None, 1e-6, 1.0, 1.0, 0.0),
    (300, 1536, "bf16", "bf16", "bf16", "feature", "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 1.0),  # rows of 192,
    (40, 2560, "f16", "f32", "f16", "token", "f16", None, 1e-6, 1e-6, 1.0, 1.0, 0.0),         # 384
    (50, 5120, "bf16", "bf16", "f32", "seq", "bf16", [20, 0, 28], 1e-6, 1e-6, 1.0, 0.5, 0.0),  # and 768 lanes
    (600, 8192, "bf16", "f32", "bf16", "feature", "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 0.0),  # two chunks a lane
    (30, 4001, "f16", "f16", "f16", "seq", "f16", [11, 0, 17], 1e-6, 1e-6, 1.0, 1.0, 0.0),    # odd rows of 512
    (300, 5003, "bf16", "bf16", "bf16", "token", "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 0.0),    # and 768 lanes
    (700, 1001, "bf16", "f32", "bf16", "feature", "bf16", None, 1e-6, 1e-6, 1.0, 1.0, 1.0),   # of 128,
    (21, 1500, "f32", "f32", "f32", "token", "f32", None, 1e-6, 1e-6, 1.0, 1.0, 0.0),         # 192
    (400, 2999, "f16", "f16", "f16", "seq", "f16", [1, 398], None, 1e-6, 1.0, 1.0, 0.0),      # and 384
    (64, 700, "f32", "f32", None, None, "f32", None, None, None, 2.0, 1.0, 0.0),         # the sum alone
    (2500, 640, "bf16", "bf16", "bf16", "seq", "bf16", [1] * 700 + [1500], None, 1e-6, 1.0, 1.0, 0.0),
]
IDS = [f"T{c[0]}-H{c[1]}-{c[2]}-{c[3]}-{c[5]}" for c in CASES]


def make(torch, case, seed=0, first=0):
    """Tensors, keywords, the gate's rows, which tokens have one, each token's sequence; `first`: where sequences start."""
    T, H, yname, xname, pname, kind, gname, lens, post_eps, pre_eps, alpha, beta, o = case
    rng = np.random.default_rng(seed)
    mk = lambda name, *s: torch.from_numpy(rng.standard_normal(s)).to(dt(torch, name)).cuda()  # noqa: E731
    x, dr, y, dh = mk(xname, T, H), mk(xname, T, H), mk(yname, T, H), mk(yname, T, H)
    kw = dict(post_eps=post_eps, pre_eps=pre_eps, alpha=alpha, beta=beta, weight_offset=o)
    if pname and post_eps is not None:
        kw["post_weight"] = mk(pname, H)
    if pname and pre_eps is not None:
        kw["pre_weight"] = mk(pname, H)
    has, seq, rows = np.ones(T, bool), None, np.ones((T, 1))
    if kind == "feature":
        kw["gate"] = mk(gname, H)
        rows = np.broadcast_to(host(kw["gate"]), (T, H))
    elif kind == "token":
        kw["gate"] = mk(gname, T, H)
        rows = host(kw["gate"])
    elif kind == "seq":
        kw["gate"] = mk(gname, len(lens), H)
        off = first + np.concatenate([[0], np.cumsum(lens)])
        kw["seq_offsets"] = torch.from_numpy(off).to(torch.int32).cuda()
        seq = np.searchsorted(off, np.arange(T), side="right") - 1
        has = (seq >= 0) & (seq < len(lens))
        seq = np.where(has, seq, 0)
        rows = np.where(has[:, None], host(kw["gate"])[seq], 0.0)
    if pre_eps is None:
        dh = None
    return x, y, dr, dh, kw, rows, has, seq


def check(torch, nat, case, made):
    T, H, yname, xname, pname, kind, gname, lens, post_eps, pre_eps, alpha, beta, o = case
    x, y, dr, dh, kw, rows, has, seq = made
    ref = Ref(host(x), host(y), rows, has, host(kw.get("post_weight")), host(kw.get("pre_weight")), post_eps, pre_eps,
              np.float64(np.float32(alpha)), np.float64(np.float32(beta)), o)
    r, h = nat.residual_norm(x, y, **kw)
    near(r, ref.r, ref.m, xname, 40, "r")
    if pre_eps is None:
        assert h is None
    else:
        near(h, ref.rh * ref.wn, ref.e * abs(ref.wn), yname, 80, "h")
    for grads in ((dr, dh), (None, dh), (dr, None)):
        if grads[0] is None and grads[1] is None:
            continue
        dx, dy, dg, dp, dn = nat.residual_norm_bwd(x, y, *grads, **kw)
        want = ref.backward(*(np.zeros((T, H)) if g is None else host(g) for g in grads))
        near(dx, *want["x"], xname, 128, "dx")
        near(dy, *want["y"], yname, 128, "dy")
        assert (dp is None, dn is None, dg is None) == ("post_weight" not in kw, "pre_weight" not in kw, kind is None)
        if dp is not None:
            near(dp, *want["wp"], pname, 128 + T, "dpost")
        if dn is not None:
            near(dn, *want["wn"], pname, 128 + T, "dpre")
        g, gm = want["gate"]
        if kind == "token":
            near(dg, g, gm, gname, 128, "dgate")
        elif kind == "feature":
            near(dg, g.sum(0), gm.sum(0), gname, 128 + T, "dgate")
        elif kind == "seq":
            a, b = np.zeros((len(lens), H)), np.zeros((len(lens), H))
            np.add.at(a, seq[has], g[has])
            np.add.at(b, seq[has], gm[has])
            near(dg, a, b, gname, 128 + T, "dgate")


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_and_backward(cuda, nat, case):
    check(cuda, nat, case, make(cuda, case))


@pytest.mark.gpu
@pytest.mark.parametrize("H,lanes,dtype,res,kind,post,pre", [
    (200, 64, "bf16", "f32", "seq", True, True), (512, 64, "f16", "f16", "token", True, True),
    (512, 64, "f32", "f32", "seq", False, True), (333, 64, "bf16", "bf16", "token", True, False),
    (1024, 128, "bf16", "bf16", "token", False, True), (1537, 256, "f16", "f16", "seq", True, True),
    (2048, 256, "bf16", "f32", "token", True, True), (2048, 256, "bf16", "bf16", None, True, True),
    (4096, 512, "bf16", "bf16", "token", True, True), (4096, 512, "f16", "f32", "feature", True, True),
    (5120, 768, "bf16", "bf16", "seq", True, True), (5120, 768, "bf16", "bf16", "token", True, True)], ids=str)
def test_several_rows_of_a_group(cuda, nat, H, lanes, dtype, res, kind, post, pre):
    """Four rows a group in the forward and more in the backward, whose rows, gates and sums pass from one to the
    next: a group of `lanes` lanes, 16 wavefronts a CU and a workgroup a CU at least.  Sequences of all lengths begin
    and end inside groups, between them tokens in none."""
    torch = cuda
    T = 3 * torch.cuda.get_device_properties(0).multi_processor_count * max(1, 16 * 64 // lanes) + 1
    lens = None
    if kind == "seq":
        rng = np.random.default_rng(5)
        lens = [0, 1, 2, 3, 4, 5, 0, 0, 9]
        while sum(lens) < T - 40:
            lens.append(int(min(T - 11 - sum(lens), np.exp(rng.uniform(0, np.log(T / 4))))))
    case = (T, H, dtype, res, dtype, kind, dtype, lens, 1e-6 if post else None, 1e-6 if pre else None, 1.0, 0.5, 1.0)
    check(torch, nat, case, make(torch, case, first=5))


@pytest.mark.gpu
def test_gradients_against_differences(cuda, nat):
    """Central differences of the forward in f32 along random directions: steps of 2^-7 leave an error of
    second order (under 1e-3 here) beside 2^-24 of the sums over 2^-7."""
    torch = cuda
    T, H = 6, 40
    g = torch.Generator("cuda").manual_seed(1)
    mk = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    p = dict(x=mk(T, H), y=mk(T, H), gate=mk(2, H), post_weight=mk(H), pre_weight=mk(H))
    off = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    dr, dh = mk(T, H), mk(T, H)

    def value(p):
        r, h = nat.residual_norm(p["x"], p["y"], gate=p["gate"], seq_offsets=off, post_weight=p["post_weight"],
                                 pre_weight=p["pre_weight"], post_eps=1e-5, pre_eps=1e-5, alpha=0.8, beta=1.3)
        return float((r.double() * dr).sum() + (h.double() * dh).sum())

    dx, dy, dg, dp, dn = nat.residual_norm_bwd(
        p["x"], p["y"], dr, dh, gate=p["gate"], seq_offsets=off, post_weight=p["post_weight"],
        pre_weight=p["pre_weight"], post_eps=1e-5, pre_eps=1e-5, alpha=0.8, beta=1.3)
    for name, grad in (("x", dx), ("y", dy), ("gate", dg), ("post_weight", dp), ("pre_weight", dn)):
        way = mk(*p[name].shape)
        way /= way.norm()
        step = 2.0 ** -7
        up, down = (value({**p, name: p[name] + s * step * way}) for s in (1, -1))
        assert abs((up - down) / (2 * step) - float((grad.double() * way).sum())) <= 1e-2 * float(grad.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_in_no_sequence(cuda, nat, dtype):
    """Tokens before the first and behind the last sequence keep r = alpha x and get dy = 0, whatever y holds there."""
    torch = cuda
    case = (40, 200, dtype, dtype, dtype, "seq", dtype, [7, 0, 11], 1e-6, 1e-6, 1.0, 1.0, 0.0)
    made = make(torch, case, first=5)
    has = made[6]
    y = made[1]
    y[torch.from_numpy(~has).cuda()] = float("nan")
    y[0] = float("inf")
    check(torch, nat, case, made)
    x, y, dr, dh, kw, *_ = made
    kw["post_eps"] = kw["pre_eps"] = 0.0
    assert torch.isfinite(nat.residual_norm(x, y, **kw)[0]).all()
    out = nat.residual_norm_bwd(x, y, dr, dh, **kw)
    assert all(torch.isfinite(t).all() for t in out)
    assert not out[1][torch.from_numpy(~has).cuda()].any()
    # No sequences at all.
    kw["gate"], kw["seq_offsets"] = kw["gate"][:0], kw["seq_offsets"][:1]
    r, _ = nat.residual_norm(x, y, **kw)
    assert torch.equal(r, x)
    out = nat.residual_norm_bwd(x, y, dr, dh, **kw)
    assert out[2].shape == (0, 200) and not out[1].any()


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_rows(cuda, nat):
    torch = cuda
    g = torch.Generator("cuda").manual_seed(2)
    x, y, dr, dh = (torch.randn(64, 300, device="cuda", generator=g) for _ in range(4))
    w = torch.ones(300, device="cuda")
    kw = dict(post_weight=w, pre_weight=w, post_eps=1e-6)
    r0, h0 = nat.residual_norm(x, y, **kw)
    d0 = nat.residual_norm_bwd(x, y, dr, dh, **kw)
    x[3, 7], y[10, 0], dr[20, 1], dh[30, 299] = float("inf"), float("nan"), float("-inf"), float("nan")
    r, h = nat.residual_norm(x, y, **kw)
    d = nat.residual_norm_bwd(x, y, dr, dh, **kw)
    clean = torch.ones(64, dtype=torch.bool, device="cuda")
    clean[[3, 10, 20, 30]] = False
    for a, b in ((r, r0), (h, h0), (d[0], d0[0]), (d[1], d0[1])):
        assert torch.equal(a[clean], b[clean])
    assert torch.isnan(h[10]).all() and torch.isnan(d[1][10]).all() and torch.isnan(d[0][30]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [256, 1201, 4096, 9000])
def test_in_place_and_strided(cuda, nat, H):
    """r over x, h over y, dx over dr, dy over dh, rows of wider tensors at any alignment: the same bits."""
    torch = cuda
    g = torch.Generator("cuda").manual_seed(3)
    T = 333
    wide = [torch.randn(T, H + 11, device="cuda", generator=g).to(torch.bfloat16) for _ in range(4)]
    keep = [t.clone() for t in wide]
    x, y, dr, dh = (t[:, 3 + k:3 + k + H] for k, t in enumerate(wide))
    w = torch.randn(H, device="cuda", generator=g)
    gate = torch.randn(T, 2 * H, device="cuda", generator=g).to(torch.float16)[:, 1:1 + H]
    kw = dict(post_weight=w, pre_weight=w, post_eps=1e-6, gate=gate)
    c = [t.clone() for t in (x, y, dr, dh)]
    r0, h0 = nat.residual_norm(c[0], c[1], **kw)
    d0 = nat.residual_norm_bwd(*c, **kw)
    d = nat.residual_norm_bwd(x, y, dr, dh, dx=dr, dy=dh, **kw)
    assert all(torch.equal(a, b) for a, b in zip(d, d0)) and d[0] is dr and d[1] is dh
    r, h = nat.residual_norm(x, y, r=x, h=y, **kw)
    assert torch.equal(r, r0) and torch.equal(h, h0)
    for k, (t, before) in enumerate(zip(wide, keep)):
        assert torch.equal(t[:, :3 + k], before[:, :3 + k]) and torch.equal(t[:, 3 + k + H:], before[:, 3 + k + H:])


@pytest.mark.gpu
def test_no_rows(cuda, nat):
    torch = cuda
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    r, h = nat.residual_norm(x, x, pre_weight=w)
    assert r.shape == h.shape == (0, 64)
    dx, dy, dg, dp, dn = nat.residual_norm_bwd(x, x, x, x, pre_weight=w, gate=w)
    assert not dn.any() and not dg.any() and dp is None
    gate = torch.ones(3, 64, device="cuda")
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert not nat.residual_norm_bwd(x, x, x, x, gate=gate, seq_offsets=off)[2].any()


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda, nat):
    """Rows a whole 2^18 elements apart in a stream of 2^32: the last rows' offsets pass 32 bits."""
    torch = cuda
    T, H, stride = 1 << 14, 64, 1 << 18
    buf = torch.zeros((T - 1) * stride + H, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (T, H), (stride, 1))
    g = torch.Generator("cuda").manual_seed(4)
    x.copy_(torch.randn(T, H, device="cuda", generator=g))
    y = torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16)
    c = x.contiguous()
    w = torch.ones(H, device="cuda")
    for a, b in zip(nat.residual_norm(x, y, pre_weight=w), nat.residual_norm(c, y, pre_weight=w)):
        assert torch.equal(a, b)
    for a, b in zip(nat.residual_norm_bwd(x, y, y, y, pre_weight=w, dx=x), nat.residual_norm_bwd(c, y, y, y, pre_weight=w)):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.gpu
def test_captured_and_on_two_streams(cuda, nat):
    torch = cuda
    case = (500, 768, "bf16", "bf16", "bf16", "seq", "bf16", [100, 0, 250, 100], 1e-6, 1e-6, 1.0, 1.0, 0.0)
    x, y, dr, dh, kw, *_ = make(torch, case)
    both = lambda: (*nat.residual_norm(x, y, **kw), *nat.residual_norm_bwd(x, y, dr, dh, **kw))  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        both()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = both()
    for k in range(4):
        kw["seq_offsets"].copy_(torch.tensor([k, 100 * k, 100 * k + 7, 400, 500 - k], dtype=torch.int32))
        x.mul_(-0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both()))
    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_refusals(nat):
    lib = nat.load()

    def fill(a, **kw):
        names = ("x", "y", "post_weight", "pre_weight", "r", "h", "dr", "dh", "dx", "dy", "dpost_weight", "dpre_weight")
        for i, f in enumerate(names):
            if hasattr(a, f):
                setattr(a, f, 0x100000 * (i + 1))
        a.T, a.H, a.alpha, a.beta, a.post_eps, a.pre_eps = 8, 64, 1.0, 1.0, 1e-6, 1e-6
        for f, _ in a._fields_:
            if f.endswith("_stride"):
                setattr(a, f, kw.get("H", 64))
        a.res_dtype = a.dtype = a.param_dtype = a.gate_dtype = nat.MFX_BF16
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    def fwd(**kw):
        return lib.mfx_residual_norm(ctypes.byref(fill(nat.ResidualNormArgs(), **kw)), None)

    def bwd(**kw):
        a = fill(nat.ResidualNormBwdArgs(), **kw)
        assert lib.mfx_residual_norm_bwd_workspace_size(ctypes.byref(a)) == 0 or "workspace" in kw
        return lib.mfx_residual_norm_bwd(ctypes.byref(a), None)

    nan = float("nan")
    for call in (fwd, bwd):
        for bad in (dict(T=-1), dict(H=0), dict(x=0), dict(y=0), dict(x=0x100001), dict(x_stride=-64), dict(alpha=nan),
                    dict(beta=float("inf")), dict(weight_offset=nan), dict(post_eps=nan), dict(pre_eps=float("inf")),
                    dict(post_eps=-1.0), dict(pre_eps=-1.0), dict(gate_mode=4), dict(gate_mode=-1), dict(num_seqs=2),
                    dict(gate_mode=1), dict(gate_mode=3, gate=0x900001), dict(gate_mode=2, num_seqs=2, gate=0x900000),
                    dict(gate_mode=2, num_seqs=-1, gate=0x900000, seq_offsets=0xa00000), dict(post_weight=0x300001)):
            assert call(**bad) == INVALID, bad
        for bad in (dict(dtype=3), dict(res_dtype=nat.MFX_F16), dict(param_dtype=9), dict(H=32769),
                    dict(gate_mode=1, gate=0x900000, gate_dtype=5), dict(T=2 ** 31)):
            assert call(**bad) == UNSUPPORTED, bad
    for bad in (dict(r=0), dict(h=0), dict(r_stride=63), dict(h=0x600001)):
        assert fwd(**bad) == INVALID, bad
    for bad in (dict(dr=0, dh=0), dict(dx=0), dict(dy=0), dict(dx_stride=63), dict(dgate=0x900000),
                dict(dh=0x800001), dict(post_weight=0), dict(pre_eps=-1.0, pre_weight=0, dpre_weight=0),
                dict(dpost_weight=0xb00001)):
        assert bwd(**bad) == INVALID, bad
    assert bwd(workspace=0xc00000, workspace_bytes=16) == WORKSPACE
    assert bwd(workspace=0xc00010, workspace_bytes=1 << 24) == INVALID
    big = dict(T=1 << 20, H=4096, gate_mode=2, num_seqs=1 << 20, gate=0x900000, dgate=0xd00000, seq_offsets=0xa00000)
    assert bwd(**big) == UNSUPPORTED and b"too large" in lib.mfx_last_error()


def test_python_checks(nat):
    torch = pytest.importorskip("torch")
    x, w = torch.zeros(4, 16), torch.zeros(16)
    off = torch.zeros(3, dtype=torch.int32)
    for kw in (dict(y=torch.zeros(4, 15)), dict(pre_weight=torch.zeros(15)), dict(pre_weight=w, post_weight=w.half(), post_eps=1e-6),
               dict(gate=torch.zeros(3, 16)), dict(gate=torch.zeros(3, 16), seq_offsets=off), dict(seq_offsets=off),
               dict(gate=torch.zeros(32)[::2]), dict(pre_eps=-1e-6), dict(post_eps=float("nan")), dict(pre_eps=None, h=x),
               dict(r=torch.zeros(4, 16, dtype=torch.float16)), dict()):  # (the last: not on a GPU)
        with pytest.raises(ValueError):
            nat.residual_norm(x, kw.pop("y", x), **kw)
    with pytest.raises(TypeError):
        nat.residual_norm(x, x, gate=torch.zeros(2, 16), seq_offsets=off.long())
    with pytest.raises(ValueError):
        nat.residual_norm_bwd(x, x, x.half(), x)
