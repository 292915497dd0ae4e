"""Calls that would need 2^32 threads or more in a launch are refused on the
host, before anything is launched, with MFX_E_UNSUPPORTED; the largest that fit
are accepted.  (No GPU needed: sizes only.)"""
import ctypes

import pytest

UNSUPPORTED = -2


@pytest.fixture(scope="module")
def nat():
    from jax_mlx_amd import native

    native.load()
    return native


def _packed(nat, bwd, T, n, Hq, Hkv, D, dtype):
    a = (nat.SdpaPackedBwdArgs if bwd else nat.SdpaPackedArgs)()
    for i, f in enumerate(("q", "k", "v", "dout", "out", "lse", "dq", "dk", "dv", "seq_offsets")):
        if hasattr(a, f):
            setattr(a, f, 0x100000 * (i + 1))
    a.T, a.num_seqs, a.Hq, a.Hkv, a.D = T, n, Hq, Hkv, D
    for f, _ in a._fields_:
        if f.endswith("_strides"):
            getattr(a, f)[:] = [D, (Hkv if f[:2] in ("k_", "v_", "dk", "dv") else Hq) * D, 1]
    a.scale, a.causal, a.dtype = 0.125, 1, dtype
    return a


# (T, sequences, Hq, Hkv, D, dtype, fits): sequences past 512 own a workgroup of
# 256 threads a head each; a row of the per-row kernels takes 64.
PACKED = [(1000, 1 << 19, 32, 8, 64, 1, False), (1000, (1 << 19) - 8, 32, 8, 64, 1, True),
          (1000, (1 << 19) - 7, 32, 8, 64, 1, False), (10, 1 << 19, 32, 8, 64, 0, False),
          (10, (1 << 24) - 1, 1, 1, 128, 2, True), (10, 1 << 24, 1, 1, 128, 2, False), (10, 1 << 20, 16, 16, 96, 1, False),
          (1 << 26, 1, 1, 1, 80, 1, False), ((1 << 26) - 4, 1, 1, 1, 80, 1, True), (1 << 21, 3, 32, 4, 72, 0, False)]


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("case", PACKED, ids=str)
def test_packed(nat, case, bwd):
    lib = nat.load()
    fn = "mfx_sdpa_packed_bwd" if bwd else "mfx_sdpa_packed"
    a = _packed(nat, bwd, *case[:-1])
    name = getattr(lib, fn + "_kernel_name")(ctypes.byref(a))
    if case[-1]:
        assert name is not None
    else:
        assert name is None and getattr(lib, fn)(ctypes.byref(a), None) == UNSUPPORTED
        assert b"too large" in lib.mfx_last_error()


def _xent(nat, bwd, T, H, V, dtype):
    a = (nat.LinearXentBwdArgs if bwd else nat.LinearXentArgs)()
    for i, f in enumerate(("h", "w", "targets", "lse", "dloss", "dh", "dw", "loss")):
        if hasattr(a, f):
            setattr(a, f, 0x100000 * (i + 1))
    a.T, a.H, a.V, a.dtype, a.target_dtype = T, H, V, dtype, nat.MFX_I64
    for f, _ in a._fields_:
        if f.endswith("_stride"):
            setattr(a, f, H)
    if bwd:
        a.dw_dtype = dtype
    return a


# Tiles of 256 x 256 (f32: 128 x 128) outputs by 256 threads; 16 threads a row.
XENT = [(1 << 20, 64, 1 << 20, 1, False), (1 << 20, 64, (1 << 20) - 256, 1, True), (1 << 20, 64, 1 << 18, 0, False),
        (1 << 20, 64, (1 << 18) - 128, 0, True), (1 << 28, 8, 10, 2, False), ((1 << 28) - 64, 8, 10, 2, True)]


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("case", XENT, ids=str)
def test_linear_xent(nat, case, bwd):
    lib = nat.load()
    fn = "mfx_linear_xent_bwd" if bwd else "mfx_linear_xent"
    a = _xent(nat, bwd, *case[:-1])
    if case[-1]:
        assert getattr(lib, fn + "_workspace_size")(ctypes.byref(a)) > 0
    else:
        assert getattr(lib, fn + "_workspace_size")(ctypes.byref(a)) == 0
        assert getattr(lib, fn)(ctypes.byref(a), None) == UNSUPPORTED and b"too large" in lib.mfx_last_error()


@pytest.mark.parametrize("B,T", [(1, 1 << 26), (1 << 13, 1 << 13)])
def test_qk_norm_rope(nat, B, T):
    """Four tokens a workgroup of 256 threads.  (The backward walks tokens in
    strides of its grid.)"""
    lib = nat.load()
    a = nat.QkNormRopeArgs()
    a.q, a.q_out, a.positions, a.freqs = 0x100000, 0x200000, 0x300000, 0x400000
    a.B, a.T, a.Hq, a.Hkv, a.D, a.rot, a.axes, a.eps, a.dtype = B, T, 1, 0, 32, 32, 1, 1e-6, nat.MFX_BF16
    a.q_strides[:] = a.qo_strides[:] = [T * 32, 32, 32, 1]
    a.sections[:] = [16, 0, 0, 0]
    assert lib.mfx_qk_norm_rope(ctypes.byref(a), None) == UNSUPPORTED and b"too large" in lib.mfx_last_error()
