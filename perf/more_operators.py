"""Workloads of the two ends of a decoder's training step and of what lies
between its blocks, through the package's public entry points
(`jax_mlx_amd.native`) where `own` is set, and in plain torch operations in 32
bits otherwise:

  embed      rows of an embedding table by token, scaled (`embedding`)
  embed_bwd  the table's gradient (`embedding_bwd`)
  norm       the norm behind a block, its gate, the residual sum and the norm
             before the next block, one pass (`residual_norm`)
  norm_bwd   the gradients of that pass (`residual_norm_bwd`)
  ortho      a stack of matrices orthogonalised by Newton-Schulz products
             (`newton_schulz`)
  muon       momentum, orthogonalisation, decay and update of a stack of weight
             matrices (`muon_update`)

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
NS_EPS = 1e-7
COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MU, DECAY = 0.02, 0.95, 0.1


def _native():
    from jax_mlx_amd import native

    return native


# ---- the cases -----------------------------------------------------------------

def listed():
    return [
        # One new token for each of 64 sequences: latency.
        dict(name="embed_decode", kind="embed", dtype="bf16", T=64, H=4096, V=65537),
        # A batch of prompts (or a training batch) of 8192 tokens, large odd vocabulary.
        dict(name="embed_prefill", kind="embed", dtype="bf16", T=8192, H=4096, V=65537),
        # The table's gradient in a small f32 model.
        dict(name="embed_grad_small", kind="embed_bwd", dtype="f32", T=257, H=512, V=1000),
        # The table's gradient of a training batch against an ordinary vocabulary.
        dict(name="embed_grad_train", kind="embed_bwd", dtype="bf16", T=16384, H=2048, V=32000),
        # One new token for each of 64 sequences, between two blocks: latency.
        dict(name="norm_decode", kind="norm", dtype="bf16", res="bf16", T=64, H=4096, post=False, pre=True,
             gate="none", params="bf16", lens=""),
        # Image patches of several pictures in one run: a gate row for each picture, a ragged number of patches.
        dict(name="norm_image", kind="norm", dtype="f16", res="f16", T=4099, H=1152, post=True, pre=True,
             gate="seq", params="f16", lens="1024,256,1,1369,777,672"),
        # A training batch's backward, residual stream in f32, a norm on both sides of the block.
        dict(name="norm_train", kind="norm_bwd", dtype="bf16", res="f32", T=8192, H=4096, post=True, pre=True,
             gate="none", params="f32", lens=""),
        # The backward with a learned scale of each feature of the block's output.
        dict(name="norm_scale_train", kind="norm_bwd", dtype="bf16", res="bf16", T=4099, H=2048, post=False, pre=True,
             gate="feature", params="bf16", lens=""),
        # One projection of a small f32 model: latency.
        dict(name="ortho_small", kind="ortho", dtype="f32", B=1, m=512, n=512),
        # The feed-forward matrices of a stack of small layers, taller than wide.
        dict(name="ortho_layers", kind="ortho", dtype="bf16", B=12, m=2048, n=512),
        # The update of a feed-forward matrix with f32 weights, ragged.
        dict(name="muon_ffn", kind="muon", dtype="f32", B=1, m=2048, n=8200, nesterov=True),
        # The update of a large square projection in bf16.
        dict(name="muon_large", kind="muon", dtype="bf16", B=1, m=4096, n=4096, nesterov=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_bwd", "embed_bwd", "norm", "norm", "norm_bwd", "norm_bwd", "ortho", "muon"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("embed", "embed_bwd"):
        H = rng.choice([8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512), _log(rng, 33, 4096)])
        V = _log(rng, 100, 65537)
        return dict(kind=kind, dtype=dtype, T=_log(rng, 1, min(32768, (1 << 25) // H)), H=H, V=V)
    if kind in ("norm", "norm_bwd"):
        H = rng.choice([8 * _log(rng, 8, 1024), 8 * _log(rng, 8, 1024), _log(rng, 33, 8192)])
        T = _log(rng, 1, min(32768, (1 << 25) // H))
        post, pre = rng.choice([(False, True), (True, True), (True, False), (True, True)])
        gate = rng.choice(["none", "none", "feature", "seq", "token"])
        lens = []
        if gate == "seq":  # lengths spread over their logarithm until the batch is full
            left = T
            while left > 0 and len(lens) < 64:
                lens.append(min(left, _log(rng, 1, T)))
                left -= lens[-1]
            lens[-1] += left
        return dict(kind=kind, dtype=dtype, res=rng.choice([dtype, dtype, "f32"]), T=T, H=H, post=post, pre=pre,
                    gate=gate, params=rng.choice([dtype, "f32"]), lens=",".join(map(str, lens)))
    m, n = _log(rng, 32, 6000), _log(rng, 32, 6000)
    if rng.random() < 0.5:
        m, n = (m + 7) // 8 * 8, (n + 7) // 8 * 8
    # At most what the largest listed case costs, and f32 at a third of its rate.
    cap = 4096 ** 3 // (3 if dtype != "bf16" else 1)
    while min(m, n) ** 2 * max(m, n) > cap:
        m, n = m * 7 // 8, n * 7 // 8
    B = rng.choice([1, 1, 2, 3, _log(rng, 1, 24)])
    B = max(1, min(B, cap // (min(m, n) ** 2 * max(m, n)), (1 << 25) // (m * n)))
    case = dict(kind=kind, dtype=dtype, B=B, m=m, n=n)
    if kind == "muon":
        case["nesterov"] = rng.random() < 0.7
    return case


# ---- inputs --------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = torch.device("cuda")
    kind, dt = case["kind"], DT[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    st = dict(case=case)
    if kind in ("embed", "embed_bwd"):
        T, H, V = case["T"], case["H"], case["V"]
        # Few tokens often and many seldom, one (the first) a twentieth of all, some that do not count.
        ids = (V * rand(T) ** 3).long().clamp_(max=V - 1)
        kinds = rand(T)
        ids = torch.where(kinds < 0.05, torch.zeros_like(ids), ids)
        st["ids"] = torch.where(kinds > 0.99, torch.full_like(ids, -100), ids)
        if kind == "embed":
            st["w"] = randn(V, H, scale=0.02)
        else:
            st["dout"] = randn(T, H)
        return st
    if kind in ("norm", "norm_bwd"):
        T, H = case["T"], case["H"]
        pdt = DT[case["params"]]
        # A residual stream that has grown over the layers, and a block's output.
        st["x"] = randn(T, H, dtype=DT[case["res"]], scale=3.0)
        st["y"] = randn(T, H)
        st["post_weight"] = (1 + randn(H, dtype=torch.float32, scale=0.2)).to(pdt) if case["post"] else None
        st["pre_weight"] = (1 + randn(H, dtype=torch.float32, scale=0.2)).to(pdt) if case["pre"] else None
        st["gate"] = st["offsets"] = st["seq"] = None
        if case["gate"] == "feature":
            st["gate"] = randn(H, dtype=pdt, scale=0.5)
        elif case["gate"] == "token":
            st["gate"] = torch.sigmoid(randn(T, H, dtype=torch.float32)).to(dt)
        elif case["gate"] == "seq":
            lens = torch.tensor([int(v) for v in case["lens"].split(",")], device=dev)
            st["gate"] = randn(lens.numel(), H, dtype=pdt, scale=0.5)
            st["offsets"] = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
            st["seq"] = torch.repeat_interleave(torch.arange(lens.numel(), device=dev), lens)
        if kind == "norm_bwd":
            st["dr"] = randn(T, H, dtype=DT[case["res"]])
            st["dh"] = randn(T, H) if case["pre"] else None
        return st
    B, m, n = case["B"], case["m"], case["n"]
    # A gradient: some directions far larger than the others.
    k = max(1, min(m, n) // 16)
    low = torch.matmul(randn(B, m, k, dtype=torch.float32), randn(B, k, n, dtype=torch.float32)) * (2.0 / k ** 0.5)
    st["g"] = ((low + torch.randn(B, m, n, generator=g, device=dev)) * 1e-3).to(dt)
    if kind == "muon":
        st["w"] = randn(B, m, n, scale=n ** -0.5)
        st["buf"] = (st["g"].float() * 0.7 + torch.randn(B, m, n, generator=g, device=dev) * 5e-4).to(dt)
    return st


# ---- the plain forms -----------------------------------------------------------

def _scale(case):
    """Of an embedding: the root of its size, as models with tied heads take it."""
    return float(case["H"]) ** 0.5


def _plain_embed(st):
    ids, w = st["ids"], st["w"]
    rows = w[ids.clamp(min=0)].float() * _scale(st["case"])
    return torch.where((ids >= 0)[:, None], rows, 0.0).to(w.dtype)


def _plain_embed_bwd(st):
    ids, case = st["ids"], st["case"]
    rows = torch.where((ids >= 0)[:, None], st["dout"].float() * _scale(case), 0.0)
    dw = torch.zeros(case["V"], case["H"], dtype=torch.float32, device=ids.device)
    return dw.index_add_(0, ids.clamp(min=0), rows).to(st["dout"].dtype)


def _alpha_beta(case):
    return (1.0, 1.0) if case["gate"] != "none" else (1.0, 0.5)


def _plain_parts(st):
    """(z, r, 1 / rms of y, of r, gate) in 32 bits."""
    alpha, beta = _alpha_beta(st["case"])
    x, y = st["x"].float(), st["y"].float()
    iy = ir = None
    z = y
    if st["post_weight"] is not None:
        iy = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        z = y * iy * st["post_weight"].float()
    gate = None if st["gate"] is None else st["gate"].float()
    if st["seq"] is not None:
        gate = gate[st["seq"]]
    r = alpha * x + beta * (z if gate is None else gate * z)
    if st["pre_weight"] is not None:
        ir = 1.0 / torch.sqrt((r * r).mean(-1, keepdim=True) + EPS)
    return z, r, iy, ir, gate


def _plain_norm(st):
    _, r, _, ir, _ = _plain_parts(st)
    h = None if ir is None else (r * ir * st["pre_weight"].float()).to(st["y"].dtype)
    return r.to(st["x"].dtype), h


def _plain_norm_bwd(st):
    alpha, beta = _alpha_beta(st["case"])
    z, r, iy, ir, gate = _plain_parts(st)
    y = st["y"].float()
    d, dpre, dpost, dgate = st["dr"].float(), None, None, None
    if ir is not None:
        rh, dh = r * ir, st["dh"].float()
        u = dh * st["pre_weight"].float()
        d = d + ir * (u - rh * (u * rh).mean(-1, keepdim=True))
        dpre = (dh * rh).sum(0).to(st["pre_weight"].dtype)
    dz = beta * d
    if gate is not None:
        dgate = dz * z
        if st["case"]["gate"] == "feature":
            dgate = dgate.sum(0)
        elif st["seq"] is not None:
            dgate = torch.zeros(st["gate"].shape, device=y.device).index_add_(0, st["seq"], dgate)
        dgate = dgate.to(st["gate"].dtype)
        dz = dz * gate
    dy = dz
    if iy is not None:
        yh, v = y * iy, dz * st["post_weight"].float()
        dy = iy * (v - yh * (v * yh).mean(-1, keepdim=True))
        dpost = (dz * yh).sum(0).to(st["post_weight"].dtype)
    return (alpha * d).to(st["x"].dtype), dy.to(st["y"].dtype), dgate, dpost, dpre


def _plain_ortho(u):
    a, b, c = COEFFS
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2).contiguous() if tall else u
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + NS_EPS)
    for _ in range(STEPS):
        s = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(1, 2) if tall else x


def _update_scale(case):
    """The update's elements at a root mean square of 0.2, whatever the matrix."""
    return 0.2 * max(case["m"], case["n"]) ** 0.5


def _plain_muon(st):
    case = st["case"]
    g, w = st["g"].float(), st["w"].float()
    buf = MU * st["buf"].float() + (1 - MU) * g
    u = (1 - MU) * g + MU * buf if case["nesterov"] else buf
    w = w * (1 - LR * DECAY) - LR * _update_scale(case) * _plain_ortho(u)
    return w.to(st["w"].dtype), buf.to(st["buf"].dtype)


# ---- one pass --------------------------------------------------------------------

def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if not own:
        if kind == "embed":
            return _plain_embed(state)
        if kind == "embed_bwd":
            return _plain_embed_bwd(state)
        if kind == "norm":
            return _plain_norm(state)
        if kind == "norm_bwd":
            return _plain_norm_bwd(state)
        if kind == "ortho":
            return _plain_ortho(state["g"].float()).to(state["g"].dtype)
        return _plain_muon(state)
    native = _native()
    if kind == "embed":
        return native.embedding(state["ids"], state["w"], scale=_scale(case))
    if kind == "embed_bwd":
        return native.embedding_bwd(state["ids"], state["dout"], case["V"], scale=_scale(case))
    if kind in ("norm", "norm_bwd"):
        alpha, beta = _alpha_beta(case)
        kw = dict(gate=state["gate"], seq_offsets=state["offsets"], post_weight=state["post_weight"],
                  pre_weight=state["pre_weight"], post_eps=EPS if case["post"] else None,
                  pre_eps=EPS if case["pre"] else None, alpha=alpha, beta=beta)
        if kind == "norm":
            return native.residual_norm(state["x"], state["y"], **kw)
        return native.residual_norm_bwd(state["x"], state["y"], state["dr"], state["dh"], **kw)
    if kind == "ortho":
        return native.newton_schulz(state["g"], steps=STEPS, coeffs=COEFFS, eps=NS_EPS)
    # (New tensors for the weights and the momentum: a pass changes none of its inputs.)
    w, buf = torch.empty_like(state["w"]), torch.empty_like(state["buf"])
    return native.muon_update(state["w"], state["g"], state["buf"], lr=LR, mu=MU, nesterov=case["nesterov"],
                              weight_decay=DECAY, scale=_update_scale(case), steps=STEPS, coeffs=COEFFS, eps=NS_EPS,
                              w_out=w, momentum_out=buf)


def work(case):
    kind, e = case["kind"], SIZE[case["dtype"]]
    if kind == "embed":  # (rows that several tokens share are read once)
        T, H, V = case["T"], case["H"], case["V"]
        return {"bytes": (T + min(T, V)) * H * e + 8 * T, "flops": T * H}
    if kind == "embed_bwd":
        T, H, V = case["T"], case["H"], case["V"]
        return {"bytes": (T + V) * H * e + 8 * T, "flops": 2 * T * H}
    if kind in ("norm", "norm_bwd"):
        n, f, p = case["T"] * case["H"], SIZE[case["res"]], SIZE[case["params"]] * case["H"]
        gate = {"none": 0, "feature": p, "seq": p * (case["lens"].count(",") + 1), "token": n * e}[case["gate"]]
        par = p * (case["post"] + case["pre"]) + gate
        if kind == "norm":  # x, y in; r, h out
            return {"bytes": 2 * n * f + n * e * (1 + case["pre"]) + par, "flops": n * (4 + 4 * case["post"] + 4 * case["pre"])}
        # x, y, dr, dh in; dx, dy out
        return {"bytes": 3 * n * f + n * e * (2 + case["pre"]) + 2 * par,
                "flops": n * (8 + 12 * case["post"] + 14 * case["pre"])}
    B, m, n = case["B"], case["m"], case["n"]
    s, l = min(m, n), max(m, n)
    # X X^T and its square are symmetric: half of each.
    flops = B * STEPS * (s * s * l + s * s * s + 2 * s * s * l)
    return {"bytes": B * m * n * e * (2 if kind == "ortho" else 5), "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------

def _exact_embed(st):
    keep = (st["ids"] >= 0).nonzero()[:, 0]
    out = torch.zeros(st["ids"].numel(), st["w"].shape[1], dtype=torch.float64, device=keep.device)
    out[keep] = st["w"].index_select(0, st["ids"][keep]).double() * math.sqrt(st["case"]["H"])
    return out


def _exact_embed_bwd(st):
    # Tokens in order, each run's sum as a difference of running sums of its own feature.
    case = st["case"]
    keep = (st["ids"] >= 0).nonzero()[:, 0]
    ids, order = torch.sort(st["ids"][keep], stable=True)
    dw = torch.zeros(case["V"], case["H"], dtype=torch.float64, device=ids.device)
    if ids.numel():
        rows = st["dout"][keep[order]].double() * math.sqrt(case["H"])
        upto = torch.cat([torch.zeros_like(rows[:1]), rows.cumsum(0)])
        tokens, count = torch.unique_consecutive(ids, return_counts=True)
        end = count.cumsum(0)
        dw[tokens] = upto[end] - upto[end - count]
    return dw


def _exact_norm(st, backward):
    case = st["case"]
    alpha, beta = _alpha_beta(case)
    x, y = st["x"].double(), st["y"].double()
    H = case["H"]
    wp, wn = (None if w is None else w.double() for w in (st["post_weight"], st["pre_weight"]))
    iy = (y.square().sum(-1, keepdim=True) / H + EPS).rsqrt() if wp is not None else None
    z = y if wp is None else y * iy * wp
    gate = torch.ones_like(y[:1]) if st["gate"] is None else st["gate"].double()
    if st["offsets"] is not None:
        t = torch.arange(case["T"], device=y.device)
        gate = gate[torch.searchsorted(st["offsets"].long(), t, right=True) - 1]
    r = alpha * x + beta * gate * z
    ir = (r.square().sum(-1, keepdim=True) / H + EPS).rsqrt() if wn is not None else None
    if not backward:
        return r, None if wn is None else r * ir * wn
    d, dpre, dpost, dgate = st["dr"].double(), None, None, None
    if wn is not None:
        u = st["dh"].double() * wn
        dpre = (st["dh"].double() * r * ir).sum(0)
        d = d + ir * u - r * ir ** 3 * ((u * r).sum(-1, keepdim=True) / H)
    if case["gate"] == "feature":
        dgate = beta * (d * z).sum(0)
    elif case["gate"] == "token":
        dgate = beta * d * z
    elif case["gate"] == "seq":
        upto = torch.nn.functional.pad((d * z).cumsum(0), (0, 0, 1, 0))
        off = st["offsets"].long()
        dgate = beta * (upto[off[1:]] - upto[off[:-1]])
    dz = beta * gate * d
    dy = dz
    if wp is not None:
        v = dz * wp
        dpost = (dz * y * iy).sum(0)
        dy = iy * v - y * iy ** 3 * ((v * y).sum(-1, keepdim=True) / H)
    return alpha * d, dy, dgate, dpost, dpre


def _exact_ortho(u):
    """By the Gram matrix of the smaller side alone: X_k = P_k X_0 (or X_0 P_k), P_k a polynomial of it."""
    a, b, c = COEFFS
    u = u / (torch.linalg.vector_norm(u, dim=(1, 2), keepdim=True) + NS_EPS)
    wide = u.shape[1] <= u.shape[2]
    s = u @ u.mT if wide else u.mT @ u
    eye = torch.eye(s.shape[1], dtype=s.dtype, device=s.device)
    p = eye.expand_as(s)
    for _ in range(STEPS):
        q = a * eye + b * s + c * (s @ s)
        p = q @ p
        s = q @ s @ q
    return p @ u if wide else u @ p


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed":
        return _exact_embed(st)
    if kind == "embed_bwd":
        return _exact_embed_bwd(st)
    if kind in ("norm", "norm_bwd"):
        return _exact_norm(st, kind == "norm_bwd")
    g = st["g"].double()
    if kind == "ortho":
        return _exact_ortho(g)
    buf = MU * st["buf"].double() + (1 - MU) * g
    u = (1 - MU) * g + MU * buf if case["nesterov"] else buf
    w = (1 - LR * DECAY) * st["w"].double() - LR * _update_scale(case) * _exact_ortho(u)
    return w, buf
