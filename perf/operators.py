"""Workloads of a decoder trained and served on packed sequences, through the
package's public entry points (`jax_mlx_amd.native`) where `own` is set, and in
plain torch operations in 32 bits (64 for angles) otherwise:

  qk        RMSNorm of each query and key head and the rotation by the token's
            position, one pass (`qk_norm_rope`): what an attention layer does
            between its projection and its attention
  qk_bwd    the gradients of that pass (`qk_norm_rope_bwd`)
  attn      attention over sequences of different lengths packed one behind
            the other, causal, with grouped heads (`sdpa_packed`)
  attn_train  the same and its gradients (`sdpa_packed_bwd`)
  loss      softmax cross entropy of a linear head, logits never stored
            (`linear_xent`)
  loss_train  the same and its gradients (`linear_xent_bwd`)

A case is a dict of plain values; `lens` is a text of sequence lengths.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

REPO = Path(__file__).resolve().parent.parent
if str(REPO / "jax-mlx-plugin_amd") not in sys.path:
    sys.path.insert(0, str(REPO / "jax-mlx-plugin_amd"))

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def _native():
    from jax_mlx_amd import native

    return native


# ---- the cases -----------------------------------------------------------------

def listed():
    return [
        # One new token for each of 64 sequences, anywhere in a long context: latency.
        dict(name="qk_decode", kind="qk", dtype="bf16", T=64, Hq=32, Hkv=8, D=128, rot=128, axes=1,
             interleaved=False, params="bf16"),
        # A batch of prompts (or a training batch) of 8192 tokens.
        dict(name="qk_prefill", kind="qk", dtype="bf16", T=8192, Hq=32, Hkv=8, D=128, rot=128, axes=1,
             interleaved=False, params="f32"),
        # Image and video patches: three position axes, a ragged number of them, pairs side by side.
        dict(name="qk_image", kind="qk", dtype="f16", T=4099, Hq=16, Hkv=16, D=96, rot=96, axes=3,
             interleaved=True, params="f32"),
        # The backward of a training step's 8192 tokens, weights' gradients included.
        dict(name="qk_train", kind="qk_bwd", dtype="bf16", T=8192, Hq=32, Hkv=8, D=128, rot=128, axes=1,
             interleaved=False, params="f32"),
        # A few short prompts of a small f32 model (8 heads of 64): latency.
        dict(name="attn_short", kind="attn", dtype="f32", Hq=8, Hkv=8, D=64, lens="1,37,128,64,5,90"),
        # A serving batch of prompts of very different lengths.
        dict(name="attn_prefill", kind="attn", dtype="bf16", Hq=32, Hkv=8, D=128,
             lens="311,4096,1,877,2048,129,1500,64,3001,17,640,256,1023,1280,733,408"),
        # Two long documents.
        dict(name="attn_long", kind="attn", dtype="bf16", Hq=32, Hkv=8, D=128, lens="4095,12289"),
        # A training batch: documents packed into 8192 tokens, forward and backward.
        dict(name="attn_train", kind="attn_train", dtype="bf16", Hq=32, Hkv=8, D=128,
             lens="1024,2500,96,700,1811,333,128,1600"),
        # The loss of a small f32 model's batch, forward and backward.
        dict(name="loss_small", kind="loss_train", dtype="f32", T=257, H=512, V=1000),
        # Scoring a handful of tokens against a large vocabulary.
        dict(name="loss_score", kind="loss", dtype="bf16", T=33, H=4096, V=65537),
        # A training batch against an ordinary vocabulary.
        dict(name="loss_train", kind="loss_train", dtype="bf16", T=4096, H=2048, V=32000),
        # A large batch against a large, odd vocabulary.
        dict(name="loss_large", kind="loss_train", dtype="bf16", T=8192, H=4096, V=65537),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qk", "qk", "qk_bwd", "attn", "attn", "attn_train", "attn_train", "loss", "loss_train",
                       "loss_train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("qk", "qk_bwd"):
        D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
        Hkv = rng.choice([1, 2, 4, 8, 8])
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        T = min(_log(rng, 1, 32768), (1 << 26) // ((Hq + Hkv) * D))
        return dict(kind=kind, dtype=dtype, T=T, Hq=Hq, Hkv=Hkv, D=D, rot=rng.choice([D, D, D, D // 4 * 2]),
                    axes=rng.choice([1, 1, 1, 2, 3]), interleaved=rng.random() < 0.3,
                    params=rng.choice([dtype, "f32"]))
    if kind in ("attn", "attn_train"):
        D = rng.choice([32, 64, 64, 96, 128, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8, 8])
        Hq = Hkv * rng.choice([1, 1, 2, 4])
        # Lengths spread over their logarithm until the batch is full, in tokens or in scores.
        total = _log(rng, 16, 16384 if dtype != "f32" else 4096)
        top = min(total, 12289)
        lens, left, pairs = [], total, 1.5e8
        while left > 0 and len(lens) < 96:
            n = min(left, _log(rng, 1, top))
            if n * n > pairs:
                break
            lens.append(n)
            left -= n
            pairs -= n * n
        return dict(kind=kind, dtype=dtype, Hq=Hq, Hkv=Hkv, D=D, lens=",".join(map(str, lens or [1])))
    H = 8 * _log(rng, 8, 512)
    V = _log(rng, 500, 65537)
    T = _log(rng, 1, 8192)
    # (f32 products run at a small part of the 16-bit rate.)
    cap = 2e12 if dtype != "f32" else 2e11
    return dict(kind=kind, dtype=dtype, T=max(1, min(T, int(cap / (H * V)))), H=H, V=V)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


# ---- inputs --------------------------------------------------------------------

def _sections(case):
    """Rotated pairs per position axis: the first axis the fewest (time), as
    image and video models share them out."""
    pairs, axes = case["rot"] // 2, case["axes"]
    if axes == 1:
        return [pairs]
    first = pairs // (2 * axes - 2) if axes > 2 else pairs // 2
    rest = pairs - first
    out = [first] + [rest // (axes - 1)] * (axes - 1)
    out[-1] += rest - (rest // (axes - 1)) * (axes - 1)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = torch.device("cuda")
    dt = DT[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    st = dict(case=case, sections=None)
    if case["kind"] in ("qk", "qk_bwd"):
        T, Hq, Hkv, D, rot, A = (case[k] for k in ("T", "Hq", "Hkv", "D", "rot", "axes"))
        # Queries, keys and values side by side, as one projection writes them.
        qkv = randn(T, Hq + 2 * Hkv, D)
        st["q"], st["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
        pdt = DT[case["params"]]
        st["qw"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(pdt)
        st["kw"] = (1 + 0.2 * torch.randn(D, generator=g, device=dev)).to(pdt)
        if A > 1:  # a video: time, then a grid
            pos = torch.randint(0, 512, (A, T), generator=g, device=dev)
        elif T <= 256:  # one token of each sequence
            pos = torch.randint(0, 1 << 20, (1, T), generator=g, device=dev)
        else:  # two sequences packed
            cut = int(torch.randint(1, T, (1,), generator=g, device=dev))
            pos = torch.cat([torch.arange(cut, device=dev), torch.arange(T - cut, device=dev)])[None]
        st["pos"] = pos.to(torch.int32).contiguous()
        st["sections"] = _sections(case)
        if case["kind"] == "qk_bwd":
            st["gq"], st["gk"] = randn(T, Hq, D), randn(T, Hkv, D)
        if own:
            st["table"] = _native().rope_table(rot, 10000.0, device=dev)
        return st
    if case["kind"] in ("attn", "attn_train"):
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        lens = _lens(case)
        T = sum(lens)
        st["lens"] = lens
        st["offsets"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        # Queries and keys as the norm and rotation leave them (rows of norm
        # about sqrt(D)), values in place in the projection's output.
        st["q"], st["k"] = randn(T, Hq, D), randn(T, Hkv, D)
        st["v"] = randn(T, Hq + 2 * Hkv, D)[:, Hq + Hkv:]
        if case["kind"] == "attn_train":
            st["g"] = randn(T, Hq, D)
        return st
    T, H, V = case["T"], case["H"], case["V"]
    st["w"] = randn(V, H, scale=H ** -0.5)
    targets = torch.randint(0, V, (T,), generator=g, device=dev)
    # A model that has learned something: the target's logit raised by 0..12.
    lift = 12 * torch.rand(T, 1, generator=g, device=dev)
    wt = st["w"][targets].float()
    st["h"] = (torch.randn(T, H, generator=g, device=dev) + lift * wt / (wt * wt).sum(-1, keepdim=True)).to(dt)
    skip = torch.rand(T, generator=g, device=dev) < 0.05
    skip[0] = False
    st["targets"] = torch.where(skip, torch.full_like(targets, -100), targets)
    st["dloss"] = torch.where(skip, 0.0, 1.0 / float((~skip).sum())).float()
    return st


# ---- the plain forms -----------------------------------------------------------

def _angles(st, rot):
    """cos, sin [T, rot/2] of each token's angles, from 64 bits."""
    dev = st["pos"].device
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device=dev),
                                   torch.tensor(st["sections"], device=dev))
    ang = st["pos"].double()[axis].t() * freq
    return torch.cos(ang).float(), torch.sin(ang).float()


def _pairs(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _unpairs(a, b, tail, interleaved):
    both = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([both, tail], -1)


def _plain_qk(st):
    case = st["case"]
    rot, il = case["rot"], case["interleaved"]
    cos, sin = _angles(st, rot)
    cos, sin = cos[:, None], sin[:, None]
    out = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        xf = x.float()
        y = xf / torch.sqrt((xf * xf).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = _pairs(y, rot, il)
        out.append(_unpairs(a * cos - b * sin, b * cos + a * sin, y[..., rot:], il).to(x.dtype))
    return tuple(out)


def _plain_qk_bwd(st):
    case = st["case"]
    rot, il = case["rot"], case["interleaved"]
    cos, sin = _angles(st, rot)
    cos, sin = cos[:, None], sin[:, None]
    grads, weights = [], []
    for x, w, g in ((st["q"], st["qw"], st["gq"]), (st["k"], st["kw"], st["gk"])):
        xf, gf = x.float(), g.float()
        r = 1.0 / torch.sqrt((xf * xf).mean(-1, keepdim=True) + EPS)
        a, b = _pairs(gf, rot, il)
        gy = _unpairs(a * cos + b * sin, b * cos - a * sin, gf[..., rot:], il)
        xh = xf * r
        gx = gy * w.float()
        weights.append((gy * xh).sum((0, 1)).to(w.dtype))
        grads.append((r * (gx - xh * (gx * xh).mean(-1, keepdim=True))).to(x.dtype))
    return (*grads, *weights)


def _plain_attn(st, train):
    case = st["case"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    G = Hq // Hkv
    scale = D ** -0.5
    outs = []
    start = 0
    for n in st["lens"]:
        sl = slice(start, start + n)
        start += n
        q, k, v = (st[x][sl].float().transpose(0, 1) for x in "qkv")
        kr, vr = (x.repeat_interleave(G, 0) if G > 1 else x for x in (k, v))
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        s = (torch.matmul(q, kr.transpose(1, 2)) * scale).masked_fill_(hidden, -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        p = s / s.sum(-1, keepdim=True)
        o = torch.matmul(p, vr)
        if not train:
            outs.append((o.transpose(0, 1),))
            continue
        g = st["g"][sl].float().transpose(0, 1)
        dv = torch.matmul(p.transpose(1, 2), g)
        ds = torch.matmul(g, vr.transpose(1, 2))
        ds = p * (ds - (g * o).sum(-1, keepdim=True)) * scale
        dq = torch.matmul(ds, kr)
        dk = torch.matmul(ds.transpose(1, 2), q)
        dk, dv = (x.view(Hkv, G, n, D).sum(1) for x in (dk, dv))
        outs.append(tuple(x.transpose(0, 1) for x in (o, dq, dk, dv)))
    out = tuple(torch.cat(x).to(st["q"].dtype) for x in zip(*outs))
    return out if train else out[0]


def _plain_loss(st, train):
    h, w = st["h"].float(), st["w"].float()
    t = st["targets"]
    valid = t >= 0
    logits = torch.matmul(h, w.t())
    top = logits.amax(-1, keepdim=True)
    picked = logits.gather(1, t.clamp(min=0)[:, None])[:, 0]
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    lse = (torch.log(total) + top)[:, 0]
    loss = torch.where(valid, lse - picked, 0.0)
    if not train:
        return loss, lse
    d = e.div_(total)
    rows = torch.arange(t.numel(), device=t.device)
    d[rows, t.clamp(min=0)] -= 1.0
    d *= torch.where(valid, st["dloss"], 0.0)[:, None]
    dh = torch.matmul(d, w)
    dw = torch.matmul(d.t(), h)
    return loss, lse, dh.to(st["h"].dtype), dw.to(st["w"].dtype)


# ---- one pass --------------------------------------------------------------------

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "qk":
            return _plain_qk(state)
        if kind == "qk_bwd":
            return _plain_qk_bwd(state)
        if kind in ("attn", "attn_train"):
            return _plain_attn(state, kind == "attn_train")
        return _plain_loss(state, kind == "loss_train")
    native = _native()
    if kind == "qk":
        return native.qk_norm_rope(state["q"], state["k"], state["pos"], state["table"], q_weight=state["qw"],
                                   k_weight=state["kw"], eps=EPS, sections=state["sections"],
                                   interleaved=case["interleaved"])
    if kind == "qk_bwd":
        return native.qk_norm_rope_bwd(state["q"], state["k"], state["gq"], state["gk"], state["pos"],
                                       state["table"], q_weight=state["qw"], k_weight=state["kw"], eps=EPS,
                                       sections=state["sections"], interleaved=case["interleaved"])
    if kind == "attn":
        return native.sdpa_packed(state["q"], state["k"], state["v"], state["offsets"], causal=True)
    if kind == "attn_train":
        q, k, v, off = state["q"], state["k"], state["v"], state["offsets"]
        lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
        out = native.sdpa_packed(q, k, v, off, causal=True, lse=lse)
        return (out, *native.sdpa_packed_bwd(q, k, v, state["g"], out, lse, off, causal=True))
    loss, lse = native.linear_xent(state["h"], state["w"], state["targets"])
    if kind == "loss":
        return loss, lse
    return (loss, lse, *native.linear_xent_bwd(state["h"], state["w"], state["targets"], lse, state["dloss"]))


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind in ("qk", "qk_bwd"):
        n = case["T"] * (case["Hq"] + case["Hkv"]) * case["D"]
        p = 2 * case["D"] * SIZE[case["params"]]
        if kind == "qk":
            return {"bytes": 2 * n * e + p + 4 * case["axes"] * case["T"], "flops": 8 * n}
        return {"bytes": 3 * n * e + 2 * p + 4 * case["axes"] * case["T"], "flops": 20 * n}
    if kind in ("attn", "attn_train"):
        lens = _lens(case)
        T, Hq, Hkv, D = sum(lens), case["Hq"], case["Hkv"], case["D"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        if kind == "attn":  # q, k, v, out; two products
            return {"bytes": 2 * T * (Hq + Hkv) * D * e, "flops": 4 * pairs * Hq * D}
        # q, k, v, dout in; out, dq, dk, dv out; seven products, scores once more in the backward
        return {"bytes": (4 * T * Hq + 4 * T * Hkv) * D * e, "flops": 14 * pairs * Hq * D}
    T, H, V = case["T"], case["H"], case["V"]
    if kind == "loss":
        return {"bytes": (T * H + V * H) * e + 16 * T, "flops": 2 * T * H * V}
    # Logits are not kept: formed for the loss and once more for the gradient.
    return {"bytes": 2 * (T * H + V * H) * e + 20 * T, "flops": 8 * T * H * V}


# ---- the definitions in 64 bits ----------------------------------------------------

def _exact_qk(st, backward):
    case = st["case"]
    rot, il, D, T = case["rot"], case["interleaved"], case["D"], case["T"]
    dev = st["q"].device
    # Each pair as a complex number, the rotation as a product with exp(i angle).
    i = torch.arange(rot // 2, device=dev)
    bounds = torch.tensor(st["sections"], device=dev).cumsum(0)
    axis = (i[:, None] >= bounds[None]).sum(1)
    angle = st["pos"].double().t()[:, axis] * torch.exp(-2.0 * i.double() / rot * math.log(10000.0))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    first = 2 * i if il else i
    second = 2 * i + 1 if il else i + rot // 2

    def rotate(y, by):
        z = torch.complex(y[..., first], y[..., second]) * by
        out = y.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    res, wts = [], []
    for name in "qk":
        x, w = st[name].double(), st[name + "w"].double()
        inv = (x.square().sum(-1, keepdim=True) / D + EPS).rsqrt()
        if not backward:
            res.append(rotate(x * inv * w, turn))
            continue
        u = rotate(st["g" + name].double(), turn.conj())
        wts.append((u * x * inv).reshape(-1, D).sum(0))
        # y = x inv w:  dx = inv (u w) - x inv^3 / D (x . u w)
        uw = u * w
        res.append(inv * uw - x * inv ** 3 * ((x * uw).sum(-1, keepdim=True) / D))
    return (*res, *wts)


def _exact_attn(st, train):
    case = st["case"]
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    off = [0]
    for n in st["lens"]:
        off.append(off[-1] + n)
    o = torch.zeros(off[-1], Hq, D, dtype=torch.float64, device=st["q"].device)
    dq = torch.zeros_like(o)
    dk = torch.zeros(off[-1], Hkv, D, dtype=torch.float64, device=o.device)
    dv = torch.zeros_like(dk)
    for a, b in zip(off, off[1:]):
        below = torch.ones(b - a, b - a, dtype=torch.bool, device=o.device).tril()
        for h in range(Hq):
            kv = h * Hkv // Hq
            q, k, v = st["q"][a:b, h].double(), st["k"][a:b, kv].double(), st["v"][a:b, kv].double()
            s = torch.where(below, q @ k.t() / math.sqrt(D), -math.inf)
            p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
            o[a:b, h] = p @ v
            if train:
                g = st["g"][a:b, h].double()
                dv[a:b, kv] += p.t() @ g
                t = p * (g @ v.t())
                ds = (t - p * t.sum(1, keepdim=True)) / math.sqrt(D)
                dq[a:b, h] = ds @ k
                dk[a:b, kv] += ds.t() @ q
    return (o, dq, dk, dv) if train else o


def _exact_loss(st, train):
    h, t = st["h"].double(), st["targets"]
    T, V = h.shape[0], st["w"].shape[0]
    w = st["w"].double()
    loss, lse = torch.zeros(T, dtype=torch.float64, device=h.device), torch.zeros(T, dtype=torch.float64, device=h.device)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for a in range(0, T, 1024):
        b = min(T, a + 1024)
        z = h[a:b] @ w.t()
        lse[a:b] = torch.logsumexp(z, 1)
        for_loss = (t[a:b] >= 0).nonzero()[:, 0]
        loss[a + for_loss] = lse[a + for_loss] - z[for_loss, t[a + for_loss]]
        if train:
            d = torch.zeros_like(z)
            d[for_loss] = torch.exp(z[for_loss] - lse[a + for_loss, None])
            d[for_loss, t[a + for_loss]] -= 1.0
            d *= st["dloss"][a:b, None].double()
            dh[a:b] = d @ w
            dw += d.t() @ h[a:b]
    return (loss, lse, dh, dw) if train else (loss, lse)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("qk", "qk_bwd"):
        return _exact_qk(st, kind == "qk_bwd")
    if kind in ("attn", "attn_train"):
        return _exact_attn(st, kind == "attn_train")
    return _exact_loss(st, kind == "loss_train")
