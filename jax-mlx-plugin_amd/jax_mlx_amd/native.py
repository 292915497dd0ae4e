"""ctypes binding of libmfx_kernels.so (the C-ABI declared in include/mfx_kernels.h).

Device memory and the current stream come from torch tensors; the arithmetic is
the library's gfx950 HIP kernels.  There is no fallback: if the library or a
GPU is missing, calls raise.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import struct
from pathlib import Path

LIB_DIR = Path(__file__).resolve().parent / "lib"
KERNELS_LIB = LIB_DIR / "libmfx_kernels.so"

MFX_F32, MFX_BF16, MFX_F16 = 0, 1, 2
MFX_I32, MFX_I64 = 3, 5
MFX_OK = 0


class MfxError(RuntimeError):
    """A libmfx_kernels.so entry point returned a non-zero code."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"mfx error {code}: {msg}")
        self.code = code


class NormArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("y", ctypes.c_void_p),
        ("gamma", ctypes.c_void_p),
        ("beta", ctypes.c_void_p),
        ("rows", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("x_row_stride", ctypes.c_int64),
        ("y_row_stride", ctypes.c_int64),
        ("eps", ctypes.c_float),
        ("dtype", ctypes.c_int32),
        ("param_dtype", ctypes.c_int32),
    ]


class NormBwdArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p),
        ("gamma", ctypes.c_void_p),
        ("dy", ctypes.c_void_p),
        ("dx", ctypes.c_void_p),
        ("dgamma", ctypes.c_void_p),
        ("dbeta", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("rows", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("x_row_stride", ctypes.c_int64),
        ("dy_row_stride", ctypes.c_int64),
        ("dx_row_stride", ctypes.c_int64),
        ("eps", ctypes.c_float),
        ("dtype", ctypes.c_int32),
        ("param_dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


I64x4 = ctypes.c_int64 * 4


class SdpaArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("q_rms_weight", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("B", ctypes.c_int64),
        ("Hq", ctypes.c_int64),
        ("Hkv", ctypes.c_int64),
        ("Tq", ctypes.c_int64),
        ("Tk", ctypes.c_int64),
        ("D", ctypes.c_int64),
        ("Dv", ctypes.c_int64),
        ("q_strides", I64x4),
        ("k_strides", I64x4),
        ("v_strides", I64x4),
        ("o_strides", I64x4),
        ("mask_strides", I64x4),
        ("scale", ctypes.c_float),
        ("q_rms_eps", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("mask_dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("lse", ctypes.c_void_p),
    ]


class SdpaBwdArgs(ctypes.Structure):
    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("dout", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("dq", ctypes.c_void_p),
        ("dk", ctypes.c_void_p),
        ("dv", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("B", ctypes.c_int64),
        ("Hq", ctypes.c_int64),
        ("Hkv", ctypes.c_int64),
        ("Tq", ctypes.c_int64),
        ("Tk", ctypes.c_int64),
        ("D", ctypes.c_int64),
        ("Dv", ctypes.c_int64),
        ("q_strides", I64x4),
        ("k_strides", I64x4),
        ("v_strides", I64x4),
        ("do_strides", I64x4),
        ("dq_strides", I64x4),
        ("dk_strides", I64x4),
        ("dv_strides", I64x4),
        ("mask_strides", I64x4),
        ("scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("mask_dtype", ctypes.c_int32),
        ("fwd_out", ctypes.c_void_p),
        ("fwd_lse", ctypes.c_void_p),
        ("fwd_out_strides", I64x4),
    ]


I64x3 = ctypes.c_int64 * 3


class SdpaPackedArgs(ctypes.Structure):
    """mfx_sdpa_packed_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "seq_offsets", "lse")]
                + [(n, ctypes.c_int64) for n in ("T", "num_seqs", "Hq", "Hkv", "D")]
                + [(n, I64x3) for n in ("q_strides", "k_strides", "v_strides", "o_strides")]
                + [("scale", ctypes.c_float)] + [(n, ctypes.c_int32) for n in ("causal", "dtype", "zero_rest")])


class SdpaPackedBwdArgs(ctypes.Structure):
    """mfx_sdpa_packed_bwd_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "dout", "out", "lse", "dq", "dk", "dv", "seq_offsets",
                                                "workspace")]
                + [("workspace_bytes", ctypes.c_size_t)]
                + [(n, ctypes.c_int64) for n in ("T", "num_seqs", "Hq", "Hkv", "D")]
                + [(n, I64x3) for n in ("q_strides", "k_strides", "v_strides", "do_strides", "o_strides",
                                        "dq_strides", "dk_strides", "dv_strides")]
                + [("scale", ctypes.c_float)] + [(n, ctypes.c_int32) for n in ("causal", "dtype", "zero_rest")])


class QkNormRopeArgs(ctypes.Structure):
    """mfx_qk_norm_rope_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "q_out", "k_out", "q_weight", "k_weight", "positions",
                                                "freqs")]
                + [(n, ctypes.c_int64) for n in ("B", "T", "Hq", "Hkv", "D", "rot")]
                + [(n, I64x4) for n in ("q_strides", "k_strides", "qo_strides", "ko_strides")]
                + [("pos_strides", ctypes.c_int64 * 3), ("sections", ctypes.c_int32 * 4)]
                + [(n, ctypes.c_int32) for n in ("axes", "interleaved", "dtype", "param_dtype")]
                + [("eps", ctypes.c_float), ("reserved", ctypes.c_int32)])


class QkNormRopeBwdArgs(ctypes.Structure):
    """mfx_qk_norm_rope_bwd_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "dq_out", "dk_out", "dq", "dk", "q_weight", "k_weight",
                                                "dq_weight", "dk_weight", "positions", "freqs", "workspace")]
                + [("workspace_bytes", ctypes.c_size_t)]
                + [(n, ctypes.c_int64) for n in ("B", "T", "Hq", "Hkv", "D", "rot")]
                + [(n, I64x4) for n in ("q_strides", "k_strides", "dqo_strides", "dko_strides", "dq_strides",
                                        "dk_strides")]
                + [("pos_strides", ctypes.c_int64 * 3), ("sections", ctypes.c_int32 * 4)]
                + [(n, ctypes.c_int32) for n in ("axes", "interleaved", "dtype", "param_dtype")]
                + [("eps", ctypes.c_float), ("reserved", ctypes.c_int32)])


class GemmArgs(ctypes.Structure):
    """mfx_gemm_args (include/mfx_kernels.h)."""

    _fields_ = [
        ("a", ctypes.c_void_p),
        ("b", ctypes.c_void_p),
        ("c", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("c_dtype", ctypes.c_int32),
        ("batch", ctypes.c_int64),
        ("m", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("k", ctypes.c_int64),
        ("lda", ctypes.c_int64),
        ("ldb", ctypes.c_int64),
        ("ldc", ctypes.c_int64),
        ("stride_a", ctypes.c_int64),
        ("stride_b", ctypes.c_int64),
        ("stride_c", ctypes.c_int64),
        ("trans_a", ctypes.c_int32),
        ("trans_b", ctypes.c_int32),
    ]


class LinearXentArgs(ctypes.Structure):
    """mfx_linear_xent_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("h", "w", "targets", "loss", "lse", "workspace")]
                + [("workspace_bytes", ctypes.c_size_t)]
                + [(n, ctypes.c_int64) for n in ("T", "H", "V", "h_stride", "w_stride")]
                + [(n, ctypes.c_int32) for n in ("dtype", "target_dtype")])


class LinearXentBwdArgs(ctypes.Structure):
    """mfx_linear_xent_bwd_args (include/mfx_kernels.h)."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("h", "w", "targets", "lse", "dloss", "dh", "dw", "workspace")]
                + [("workspace_bytes", ctypes.c_size_t)]
                + [(n, ctypes.c_int64) for n in ("T", "H", "V", "h_stride", "w_stride", "dh_stride", "dw_stride")]
                + [(n, ctypes.c_int32) for n in ("dtype", "target_dtype", "dw_dtype", "reserved")])


MFX_MAX_RANK = 8
MFX_EW_MAX_INPUTS = 8
MFX_EW_MAX_INSTRS = 64

# Elementwise opcodes (enum order of include/mfx_kernels.h).
EW_OPS = ["load", "const", "iota", "neg", "abs", "exp", "expm1", "log", "log1p", "sqrt", "rsqrt", "tanh",
          "logistic", "erf", "sin", "cos", "floor", "ceil", "round_ne", "sign", "not", "round_bf16",
          "round_f16", "to_int", "is_finite", "copy", "add", "sub", "mul", "div", "max", "min", "pow", "rem",
          "and", "or", "xor", "eq", "ne", "lt", "le", "gt", "ge", "atan2", "select", "clamp"]
EW_OP = {name: i for i, name in enumerate(EW_OPS)}


class EwInstr(ctypes.Structure):
    _fields_ = [("op", ctypes.c_uint8), ("dst", ctypes.c_uint8), ("a", ctypes.c_uint8), ("b", ctypes.c_uint8),
                ("c", ctypes.c_uint8), ("flags", ctypes.c_uint8), ("pad", ctypes.c_uint8 * 2),
                ("imm", ctypes.c_float)]


class EwInput(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("pad", ctypes.c_int32),
                ("strides", ctypes.c_int64 * MFX_MAX_RANK)]


class EwProgram(ctypes.Structure):
    """mfx_ew_program (include/mfx_kernels.h)."""

    _fields_ = [("out", ctypes.c_void_p), ("out_dtype", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("dims", ctypes.c_int64 * MFX_MAX_RANK), ("out_strides", ctypes.c_int64 * MFX_MAX_RANK),
                ("num_inputs", ctypes.c_int32), ("num_instrs", ctypes.c_int32), ("result", ctypes.c_int32),
                ("pad", ctypes.c_int32), ("inputs", EwInput * MFX_EW_MAX_INPUTS),
                ("code", EwInstr * MFX_EW_MAX_INSTRS)]


def ew_program(dims, inputs, code, result, out_dtype=MFX_F32):
    """Builds an EwProgram.  inputs: [(dtype_code, strides)] (data pointers
    are set by the caller); code: [(op_name, dst, a, b, c, imm)] with
    trailing fields optional (0, and imm 0.0); result: register of the
    output."""
    p = EwProgram()
    p.out_dtype = out_dtype
    p.rank = len(dims)
    for d, x in enumerate(dims):
        p.dims[d] = x
    p.num_inputs = len(inputs)
    for i, (dt, strides) in enumerate(inputs):
        p.inputs[i].dtype = dt
        for d, x in enumerate(strides):
            p.inputs[i].strides[d] = x
    p.num_instrs = len(code)
    for pc, ins in enumerate(code):
        op, dst, *rest = ins
        a, b, c, imm = list(rest) + [0, 0, 0, 0.0][len(rest):]
        p.code[pc].op = EW_OP[op]
        p.code[pc].dst = dst
        p.code[pc].a = a
        p.code[pc].b = b
        p.code[pc].c = c
        p.code[pc].imm = imm
    p.result = result
    return p


_lib = None


def load(path: str | os.PathLike | None = None, make_default: bool = False) -> ctypes.CDLL:
    """Loads libmfx_kernels.so (once) and declares its signatures.  A `path`
    loads that copy instead (for example the phase-timer build); with
    make_default the module's calls use it from then on."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else KERNELS_LIB
    if not p.exists():
        raise FileNotFoundError(
            f"{p} is not built; run `python jax-mlx-plugin_amd/build.py` (or __graft_entry__.build())")
    lib = ctypes.CDLL(str(p))
    lib.mfx_last_error.restype = ctypes.c_char_p
    lib.mfx_version.restype = ctypes.c_int
    lib.mfx_device_count.restype = ctypes.c_int
    for name in ("mfx_layer_norm", "mfx_rms_norm", "mfx_softmax", "mfx_log_softmax"):
        fn = getattr(lib, name)
        fn.argtypes = [ctypes.POINTER(NormArgs), ctypes.c_void_p]
        fn.restype = ctypes.c_int
    lib.mfx_layer_norm_bwd.argtypes = [ctypes.POINTER(NormBwdArgs), ctypes.c_void_p]
    lib.mfx_layer_norm_bwd.restype = ctypes.c_int
    lib.mfx_layer_norm_bwd_workspace_size.argtypes = [ctypes.POINTER(NormBwdArgs)]
    lib.mfx_layer_norm_bwd_workspace_size.restype = ctypes.c_size_t
    lib.mfx_sdpa_bwd.argtypes = [ctypes.POINTER(SdpaBwdArgs), ctypes.c_void_p]
    lib.mfx_sdpa_bwd.restype = ctypes.c_int
    lib.mfx_sdpa_bwd_workspace_size.argtypes = [ctypes.POINTER(SdpaBwdArgs)]
    lib.mfx_sdpa_bwd_workspace_size.restype = ctypes.c_size_t
    lib.mfx_sdpa_bwd_kernel_name.argtypes = [ctypes.POINTER(SdpaBwdArgs)]
    lib.mfx_sdpa_bwd_kernel_name.restype = ctypes.c_char_p
    lib.mfx_sdpa_fwd.argtypes = [ctypes.POINTER(SdpaArgs), ctypes.c_void_p]
    lib.mfx_sdpa_fwd.restype = ctypes.c_int
    lib.mfx_sdpa_fwd_noalloc.argtypes = [ctypes.POINTER(SdpaArgs), ctypes.c_void_p]
    lib.mfx_sdpa_fwd_noalloc.restype = ctypes.c_int
    lib.mfx_sdpa_workspace_size.argtypes = [ctypes.POINTER(SdpaArgs)]
    lib.mfx_sdpa_workspace_size.restype = ctypes.c_size_t
    lib.mfx_sdpa_kernel_name.argtypes = [ctypes.POINTER(SdpaArgs)]
    lib.mfx_sdpa_kernel_name.restype = ctypes.c_char_p
    for name, args in (("mfx_linear_xent", LinearXentArgs), ("mfx_linear_xent_bwd", LinearXentBwdArgs)):
        getattr(lib, name).argtypes = [ctypes.POINTER(args), ctypes.c_void_p]
        getattr(lib, name).restype = ctypes.c_int
        getattr(lib, name + "_workspace_size").argtypes = [ctypes.POINTER(args)]
        getattr(lib, name + "_workspace_size").restype = ctypes.c_size_t
    for name, args in (("mfx_sdpa_packed", SdpaPackedArgs), ("mfx_sdpa_packed_bwd", SdpaPackedBwdArgs)):
        getattr(lib, name).argtypes = [ctypes.POINTER(args), ctypes.c_void_p]
        getattr(lib, name).restype = ctypes.c_int
        getattr(lib, name + "_kernel_name").argtypes = [ctypes.POINTER(args)]
        getattr(lib, name + "_kernel_name").restype = ctypes.c_char_p
    lib.mfx_sdpa_packed_bwd_workspace_size.argtypes = [ctypes.POINTER(SdpaPackedBwdArgs)]
    lib.mfx_sdpa_packed_bwd_workspace_size.restype = ctypes.c_size_t
    lib.mfx_rope_freqs.argtypes = [ctypes.c_double, ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]
    lib.mfx_rope_freqs.restype = ctypes.c_int
    lib.mfx_qk_norm_rope.argtypes = [ctypes.POINTER(QkNormRopeArgs), ctypes.c_void_p]
    lib.mfx_qk_norm_rope.restype = ctypes.c_int
    lib.mfx_qk_norm_rope_bwd.argtypes = [ctypes.POINTER(QkNormRopeBwdArgs), ctypes.c_void_p]
    lib.mfx_qk_norm_rope_bwd.restype = ctypes.c_int
    lib.mfx_qk_norm_rope_bwd_workspace_size.argtypes = [ctypes.POINTER(QkNormRopeBwdArgs)]
    lib.mfx_qk_norm_rope_bwd_workspace_size.restype = ctypes.c_size_t
    lib.mfx_gemm.argtypes = [ctypes.POINTER(GemmArgs), ctypes.c_void_p]
    lib.mfx_gemm.restype = ctypes.c_int
    lib.mfx_gemm_kernel_name.argtypes = [ctypes.POINTER(GemmArgs)]
    lib.mfx_gemm_kernel_name.restype = ctypes.c_char_p
    lib.mfx_gemm_ew.argtypes = [ctypes.POINTER(GemmArgs), ctypes.POINTER(EwProgram), ctypes.c_int, ctypes.c_void_p]
    lib.mfx_gemm_ew.restype = ctypes.c_int
    lib.mfx_gemm_ew_check.argtypes = [ctypes.POINTER(GemmArgs), ctypes.POINTER(EwProgram), ctypes.c_int]
    lib.mfx_gemm_ew_check.restype = ctypes.c_int
    lib.mfx_gemm_ew_prepare.argtypes = [ctypes.POINTER(GemmArgs), ctypes.POINTER(EwProgram), ctypes.c_int]
    lib.mfx_gemm_ew_prepare.restype = ctypes.c_int
    lib.mfx_gemm_ew_source.argtypes = [ctypes.POINTER(GemmArgs), ctypes.POINTER(EwProgram), ctypes.c_int,
                                       ctypes.c_char_p, ctypes.c_int64]
    lib.mfx_gemm_ew_source.restype = ctypes.c_int64
    lib.mfx_elementwise.argtypes = [ctypes.POINTER(EwProgram), ctypes.c_void_p]
    lib.mfx_elementwise.restype = ctypes.c_int
    if path is None or make_default:
        _lib = lib
    return lib


def check(rc: int) -> None:
    if rc != MFX_OK:
        raise MfxError(rc, load().mfx_last_error().decode())


# ---- torch plumbing ------------------------------------------------------------

# A small call spends more time here than on the GPU, so the wrappers keep to
# what a call needs: structs filled by position, dtypes from a table, no views
# made to read a stride.  (A LayerNorm of [1024, 512] went from 11.0 to 9.1 us
# a call, an f32 attention of [8, 8, 128, 64] from 12.6 to 10.7.)

_torch_mod = None
_DTYPE_CODES: dict = {}


def _torch():
    global _torch_mod
    if _torch_mod is None:
        import torch  # noqa: PLC0415

        _DTYPE_CODES.update({torch.float32: MFX_F32, torch.bfloat16: MFX_BF16, torch.float16: MFX_F16})
        _torch_mod = torch
    return _torch_mod


def dtype_code(dt) -> int:
    _torch()
    code = _DTYPE_CODES.get(dt)
    if code is None:
        raise TypeError(f"unsupported dtype {dt}")
    return code


def _stream_handle(t) -> int:
    return _torch().cuda.current_stream(t.device).cuda_stream


def _require_gpu(*ts) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tensor must live on the GPU (device memory)")


def _rows_view(x):
    """(rows, n, row_stride) of a tensor whose last dim is contiguous and whose
    leading dims collapse to one row index."""
    if x.dim() == 0:
        raise ValueError("scalar input")
    n = x.shape[-1]
    if x.stride(-1) != 1:
        raise ValueError("last dimension must be contiguous")
    rows = x.numel() // n if n else 0
    if x.dim() == 1:
        return 1, n, n
    if rows > 1 and x.is_contiguous():
        return rows, n, n
    lead = x.reshape(-1, n) if x.is_contiguous() else None
    if lead is None:
        # Leading dims must still collapse with a single stride.
        try:
            lead = x.view(-1, n)
        except RuntimeError as e:
            raise ValueError("leading dimensions must collapse to one row stride") from e
    return rows, n, lead.stride(0)


def _norm_call(fn_name, x, gamma, beta, eps, out):
    torch = _torch()
    _require_gpu(x, gamma, beta)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows, n, xs = _rows_view(x)
    _, _, ys = _rows_view(out)
    dt = dtype_code(x.dtype)
    p = gamma if gamma is not None else beta
    a = NormArgs(x.data_ptr(), out.data_ptr(), gamma.data_ptr() if gamma is not None else None,
                 beta.data_ptr() if beta is not None else None, rows, n, xs, ys, float(eps), dt,
                 dtype_code(p.dtype) if p is not None else dt)
    check(getattr(load(), fn_name)(ctypes.byref(a), _stream_handle(x)))
    return out


def layer_norm(x, gamma=None, beta=None, eps: float = 1e-5, out=None):
    """(x - mean) / sqrt(var + eps) * gamma + beta over the last axis (mfx_layer_norm)."""
    return _norm_call("mfx_layer_norm", x, gamma, beta, eps, out)


def rms_norm(x, weight=None, eps: float = 1e-5, out=None):
    """x / sqrt(mean(x^2) + eps) * weight over the last axis (mfx_rms_norm)."""
    return _norm_call("mfx_rms_norm", x, weight, None, eps, out)


def softmax(x, out=None):
    """Softmax over the last axis (mfx_softmax)."""
    return _norm_call("mfx_softmax", x, None, None, 0.0, out)


def log_softmax(x, out=None):
    """Log-softmax over the last axis (mfx_log_softmax)."""
    return _norm_call("mfx_log_softmax", x, None, None, 0.0, out)


def layer_norm_bwd(x, dy, gamma=None, eps: float = 1e-5, *, param_grads=True, param_dtype=None,
                   dx=None, workspace=None):
    """(dx, dgamma, dbeta) of LayerNorm over the last axis (mfx_layer_norm_bwd).

    dgamma / dbeta have gamma's dtype (or `param_dtype`, default x's dtype when
    gamma is None); with param_grads=False only dx is computed."""
    torch = _torch()
    _require_gpu(x, dy, gamma)
    if dx is None:
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows, n, xs = _rows_view(x)
    _, _, gs = _rows_view(dy)
    _, _, ds = _rows_view(dx)
    pdt = gamma.dtype if gamma is not None else (param_dtype or x.dtype)
    dg = db = None
    if param_grads:
        dg = torch.empty(n, dtype=pdt, device=x.device)
        db = torch.empty(n, dtype=pdt, device=x.device)
    a = NormBwdArgs(x.data_ptr(), gamma.data_ptr() if gamma is not None else None, dy.data_ptr(), dx.data_ptr(),
                    dg.data_ptr() if dg is not None else None, db.data_ptr() if db is not None else None, None, 0,
                    rows, n, xs, gs, ds, float(eps), dtype_code(x.dtype), dtype_code(pdt))
    if workspace is not None:
        a.workspace = workspace.data_ptr()
        a.workspace_bytes = workspace.numel() * workspace.element_size()
    check(load().mfx_layer_norm_bwd(ctypes.byref(a), _stream_handle(x)))
    return dx, dg, db


def layer_norm_bwd_workspace_size(x, gamma=None, param_grads=True) -> int:
    """Bytes of workspace mfx_layer_norm_bwd needs (host-only query)."""
    rows, n, xs = _rows_view(x)
    a = NormBwdArgs(x=16, dy=16, dx=16, dgamma=16 if param_grads else None,
                    dbeta=16 if param_grads else None, rows=rows, n=n, x_row_stride=xs,
                    dy_row_stride=n, dx_row_stride=n, eps=1e-5, dtype=dtype_code(x.dtype),
                    param_dtype=dtype_code(gamma.dtype if gamma is not None else x.dtype))
    return int(load().mfx_layer_norm_bwd_workspace_size(ctypes.byref(a)))


def _strides4(t, layout: str):
    s = t.stride()
    if layout == "bhtd":
        return (s[0], s[1], s[2], s[3])
    if layout == "bthd":
        return (s[0], s[2], s[1], s[3])
    raise ValueError(f"layout must be 'bhtd' or 'bthd', got {layout!r}")


def _dims(t, layout):
    if layout == "bhtd":
        return t.shape[0], t.shape[1], t.shape[2], t.shape[3]
    return t.shape[0], t.shape[2], t.shape[1], t.shape[3]


# The two argument structs as one packing each (native alignment), in field
# order: a ctypes struct filled field by field takes several times as long.
_SDPA_PACK = struct.Struct("7PN7q20q2f4iP").pack
_SDPA_BWD_PACK = struct.Struct("9PN7q32qf3i2P4q").pack


def _mask_fields(mask):
    """(pointer, [B, H, Tq, Tk] strides, dtype code) of an additive mask
    (broadcast dims, of size 1, get stride 0); nulls for None."""
    if mask is None:
        return 0, (0, 0, 0, 0), 0
    strides = tuple([0 if n == 1 else st for n, st in zip(mask.shape, mask.stride())])
    return mask.data_ptr(), ((0,) * (4 - len(strides)) + strides)[:4], dtype_code(mask.dtype)


def _f32(x):
    """x as a C float holds it (past the range: an infinity, which packing refuses to make)."""
    return ctypes.c_float(x).value


def sdpa_args(q, k, v, out, *, scale=None, causal=False, mask=None, layout="bhtd",
              q_rms_eps=None, q_rms_weight=None, workspace=None, lse=None) -> SdpaArgs:
    B, Hq, Tq, D = _dims(q, layout)
    _, Hkv, Tk, _ = _dims(k, layout)
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    if mask is not None and mask.dim() > 4:
        raise ValueError("mask must have at most 4 dims [B, H, Tq, Tk]")
    mp, ms, md = _mask_fields(mask)
    if lse is not None and (lse.dtype != _torch().float32 or lse.numel() != B * Hq * Tq or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous f32 tensor of B * Hq * Tq elements")
    return SdpaArgs.from_buffer_copy(_SDPA_PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), mp,
        q_rms_weight.data_ptr() if q_rms_weight is not None else 0,
        workspace.data_ptr() if workspace is not None else 0,
        workspace.numel() * workspace.element_size() if workspace is not None else 0,
        B, Hq, Hkv, Tq, Tk, D, v.shape[-1], *_strides4(q, layout), *_strides4(k, layout), *_strides4(v, layout),
        *_strides4(out, layout), *ms, _f32(scale), _f32(q_rms_eps) if q_rms_eps is not None else -1.0,
        1 if causal else 0, dtype_code(q.dtype), md, 0, lse.data_ptr() if lse is not None else 0))


def sdpa(q, k, v, *, scale=None, causal=False, mask=None, layout="bhtd", q_rms_eps=None,
         q_rms_weight=None, out=None, workspace=None, lse=None):
    """softmax(scale * Q K^T + mask) V (mfx_sdpa_fwd).

    layout "bhtd": q [B,Hq,Tq,D], k/v [B,Hkv,Tk,D]; "bthd": JAX's BTNH layout.
    lse: optional f32 [B * Hq * Tq] output of the row log-sum-exp (log2
    units), for sdpa_bwd(fwd_out=..., fwd_lse=...).
    """
    torch = _torch()
    _require_gpu(q, k, v, mask, q_rms_weight)
    if out is None:
        shape = list(q.shape)
        shape[-1] = v.shape[-1]
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    a = sdpa_args(q, k, v, out, scale=scale, causal=causal, mask=mask, layout=layout,
                  q_rms_eps=q_rms_eps, q_rms_weight=q_rms_weight, workspace=workspace, lse=lse)
    check(load().mfx_sdpa_fwd(ctypes.byref(a), _stream_handle(q)))
    return out


def sdpa_noalloc(q, k, v, out, *, scale=None, causal=False, mask=None, layout="bhtd", q_rms_eps=None,
                 q_rms_weight=None):
    """sdpa() through mfx_sdpa_fwd_noalloc: no device allocation, the
    workspace is the library's static per-device scratch (at most
    NOALLOC_SCRATCH_BYTES); the caller passes `out`."""
    _require_gpu(q, k, v, out, mask, q_rms_weight)
    a = sdpa_args(q, k, v, out, scale=scale, causal=causal, mask=mask, layout=layout,
                  q_rms_eps=q_rms_eps, q_rms_weight=q_rms_weight)
    check(load().mfx_sdpa_fwd_noalloc(ctypes.byref(a), _stream_handle(q)))
    return out


NOALLOC_SCRATCH_BYTES = 16 << 20  # MFX_SDPA_NOALLOC_SCRATCH_BYTES


def sdpa_workspace_size(q, k, v, **kw) -> int:
    """Bytes of workspace mfx_sdpa_fwd needs for these tensors (host-only)."""
    out = kw.pop("out", None)
    a = sdpa_args(q, k, v, out if out is not None else q, **kw)
    return int(load().mfx_sdpa_workspace_size(ctypes.byref(a)))


def sdpa_kernel_name(q, k, v, **kw) -> str:
    """Which kernel mfx_sdpa_fwd picks for these tensors (host-only query)."""
    out = kw.pop("out", None)
    a = sdpa_args(q, k, v, out if out is not None else q, **kw)
    name = load().mfx_sdpa_kernel_name(ctypes.byref(a))
    if name is None:
        raise MfxError(-1, load().mfx_last_error().decode())
    return name.decode()


def sdpa_bwd_args(q, k, v, dout, dq, dk, dv, *, scale=None, causal=False, mask=None, layout="bhtd",
                  workspace=None, fwd_out=None, fwd_lse=None) -> SdpaBwdArgs:
    B, Hq, Tq, D = _dims(q, layout)
    _, Hkv, Tk, _ = _dims(k, layout)
    if scale is None:
        scale = 1.0 / (D ** 0.5)
    mp, ms, md = _mask_fields(mask)
    return SdpaBwdArgs.from_buffer_copy(_SDPA_BWD_PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(), mp, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
        workspace.data_ptr() if workspace is not None else 0,
        workspace.numel() * workspace.element_size() if workspace is not None else 0,
        B, Hq, Hkv, Tq, Tk, D, v.shape[-1], *_strides4(q, layout), *_strides4(k, layout), *_strides4(v, layout),
        *_strides4(dout, layout), *_strides4(dq, layout), *_strides4(dk, layout), *_strides4(dv, layout), *ms,
        _f32(scale), 1 if causal else 0, dtype_code(q.dtype), md,
        fwd_out.data_ptr() if fwd_out is not None else 0, fwd_lse.data_ptr() if fwd_lse is not None else 0,
        *(_strides4(fwd_out, layout) if fwd_out is not None else (0, 0, 0, 0))))


def sdpa_bwd(q, k, v, dout, *, scale=None, causal=False, mask=None, layout="bhtd", workspace=None,
             fwd_out=None, fwd_lse=None):
    """(dq, dk, dv) of softmax(scale * Q K^T + mask) V for upstream gradient dout
    (mfx_sdpa_bwd); layouts as sdpa().  fwd_out / fwd_lse: the forward call's
    output and lse on the same inputs (both or neither) to skip the
    recomputed forward pass."""
    torch = _torch()
    _require_gpu(q, k, v, dout, mask, fwd_out, fwd_lse)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    a = sdpa_bwd_args(q, k, v, dout, dq, dk, dv, scale=scale, causal=causal, mask=mask, layout=layout,
                      workspace=workspace, fwd_out=fwd_out, fwd_lse=fwd_lse)
    check(load().mfx_sdpa_bwd(ctypes.byref(a), _stream_handle(q)))
    return dq, dk, dv


def sdpa_bwd_kernel_name(q, k, v, **kw) -> str:
    """Which backward kernels mfx_sdpa_bwd picks (host-only query) for outputs
    of their own."""
    a = sdpa_bwd_args(q, k, v, q, q, k, v, **kw)
    a.dq = a.dk = a.dv = 256  # (apart from the inputs, 16-byte aligned)
    name = load().mfx_sdpa_bwd_kernel_name(ctypes.byref(a))
    if name is None:
        raise MfxError(-1, load().mfx_last_error().decode())
    return name.decode()


def sdpa_bwd_workspace_size(q, k, v, **kw) -> int:
    a = sdpa_bwd_args(q, k, v, q, q, k, v, **kw)
    return int(load().mfx_sdpa_bwd_workspace_size(ctypes.byref(a)))


# ---- helpers of the operators below ----------------------------------------------

_HERE = contextlib.nullcontext()


def _on(t, *others):
    """Context in which work for t's device is launched: t's device made the
    current one if it is not.  The other tensors (or None) must live there too."""
    index = t.get_device()
    if index < 0:
        raise ValueError("tensor must live on the GPU (device memory)")
    for o in others:
        if o is not None and o.get_device() != index:
            raise ValueError(f"tensors on {t.device} and {o.device}: all must live on one GPU")
    if _torch().cuda.current_device() == index:
        return _HERE
    return _torch().cuda.device(index)


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _fresh(t):
    """A new contiguous tensor like t (None for None)."""
    if t is None:
        return None
    return _torch().empty_like(t, memory_format=_torch().contiguous_format)


def _workspace(a, query, workspace, like):
    """Sets a.workspace: the caller's, or one from torch's allocator for this
    call (also inside a captured graph, whose pool then owns it)."""
    if workspace is None:
        need = int(getattr(load(), query)(ctypes.byref(a)))
        if not need:
            return None
        workspace = _torch().empty(need, dtype=_torch().uint8, device=like.device)
    a.workspace = workspace.data_ptr()
    a.workspace_bytes = workspace.numel() * workspace.element_size()
    return workspace


# ---- packed sequences ------------------------------------------------------------

_PACKED_PACK = struct.Struct("6P5q12qf3i").pack
_PACKED_BWD_PACK = struct.Struct("11PN5q24qf3i").pack


def _packed_dims(q, k, v, seq_offsets, *like_q):
    """(T, sequences, Hq, Hkv, D) of checked [T, H, D] tensors."""
    shape, dt, ks = q.shape, q.dtype, k.shape
    if len(shape) != 3 or len(ks) != 3:
        raise ValueError("packed q, k and v are [T, heads, head size]")
    T, Hq, D = shape
    if ks != v.shape or ks[0] != T or ks[2] != D:
        raise ValueError("k and v must agree with each other and with q in tokens and head size")
    if k.dtype != dt or v.dtype != dt:
        raise ValueError("packed tensors must share one dtype")
    for t in like_q:
        if t.shape != shape or t.dtype != dt:
            raise ValueError("out and the gradients must have q's shape and dtype")
    if seq_offsets.dtype != _torch().int32 or seq_offsets.dim() != 1 or not seq_offsets.is_contiguous():
        raise TypeError("seq_offsets must be a contiguous int32 vector")
    n = seq_offsets.numel()
    if n < 1:
        raise ValueError("seq_offsets has one more entry than there are sequences")
    return T, n - 1, Hq, ks[1], D


def _htd(t):
    s = t.stride()
    return s[1], s[0], s[2]


def _packed_lse(lse, Hq, T):
    if lse.dtype != _torch().float32 or lse.numel() != Hq * T or not lse.is_contiguous():
        raise ValueError("lse must be a contiguous f32 tensor of [heads, tokens]")


def sdpa_packed_args(q, k, v, out, seq_offsets, *, scale=None, causal=True, lse=None, zero_rest=0) -> SdpaPackedArgs:
    dims = _packed_dims(q, k, v, seq_offsets, out)
    if lse is not None:
        _packed_lse(lse, dims[2], dims[0])
    return SdpaPackedArgs.from_buffer_copy(_PACKED_PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), seq_offsets.data_ptr(), _ptr(lse), *dims, *_htd(q),
        *_htd(k), *_htd(v), *_htd(out), _f32(1.0 / (dims[4] ** 0.5) if scale is None else scale), 1 if causal else 0,
        dtype_code(q.dtype), zero_rest))


def sdpa_packed(q, k, v, seq_offsets, *, scale=None, causal=True, out=None, lse=None):
    """Attention over packed sequences (mfx_sdpa_packed): q [T, Hq, D], k and v
    [T, Hkv, D], sequence s the tokens seq_offsets[s] .. seq_offsets[s + 1]
    (int32, on the device).  Rows in no sequence are zeros in an out made here;
    a given out keeps its own there (and what takes it next goes over every
    row: they should be finite).  lse: optional f32 [Hq, T] output for
    sdpa_packed_bwd."""
    made = out is None
    if made:
        out = _fresh(q)
    a = sdpa_packed_args(q, k, v, out, seq_offsets, scale=scale, causal=causal, lse=lse, zero_rest=1 if made else 0)
    with _on(q, k, v, out, seq_offsets, lse):
        check(load().mfx_sdpa_packed(ctypes.byref(a), _stream_handle(q)))
    return out


def sdpa_packed_kernel_name(q, k, v, seq_offsets, **kw) -> str:
    """Which kernel mfx_sdpa_packed picks for these tensors (host-only query)."""
    name = load().mfx_sdpa_packed_kernel_name(ctypes.byref(sdpa_packed_args(q, k, v, q, seq_offsets, **kw)))
    if name is None:
        raise MfxError(-1, load().mfx_last_error().decode())
    return name.decode()


def sdpa_packed_bwd_args(q, k, v, dout, out, lse, dq, dk, dv, seq_offsets, *, scale=None, causal=True,
                         zero_rest=0) -> SdpaPackedBwdArgs:
    dims = _packed_dims(q, k, v, seq_offsets, dout, out, dq)
    _packed_lse(lse, dims[2], dims[0])
    if dk.shape != k.shape or dv.shape != v.shape or dk.dtype != q.dtype or dv.dtype != q.dtype:
        raise ValueError("dk and dv must match k and v")
    return SdpaPackedBwdArgs.from_buffer_copy(_PACKED_BWD_PACK(
        *[t.data_ptr() for t in (q, k, v, dout, out, lse, dq, dk, dv, seq_offsets)], 0, 0, *dims,
        *[x for t in (q, k, v, dout, out, dq, dk, dv) for x in _htd(t)],
        _f32(1.0 / (dims[4] ** 0.5) if scale is None else scale), 1 if causal else 0, dtype_code(q.dtype), zero_rest))


def sdpa_packed_bwd(q, k, v, dout, out, lse, seq_offsets, *, scale=None, causal=True, dq=None, dk=None, dv=None,
                    workspace=None):
    """(dq, dk, dv) of sdpa_packed for the gradient dout of its output, from
    its out and lse (mfx_sdpa_packed_bwd).  Rows in no sequence are zeros in
    the gradients made here; given ones keep their own there (which a sum over
    every row, as qk_norm_rope_bwd's for its weights, takes in)."""
    made = (1 if dq is None else 0) | (2 if dk is None else 0) | (4 if dv is None else 0)
    dq, dk, dv = (_fresh(t) if g is None else g for t, g in ((q, dq), (k, dk), (v, dv)))
    a = sdpa_packed_bwd_args(q, k, v, dout, out, lse, dq, dk, dv, seq_offsets, scale=scale, causal=causal,
                             zero_rest=made)
    with _on(q, k, v, dout, out, lse, dq, dk, dv, seq_offsets, workspace):
        keep = _workspace(a, "mfx_sdpa_packed_bwd_workspace_size", workspace, q)  # noqa: F841 (until the launch)
        check(load().mfx_sdpa_packed_bwd(ctypes.byref(a), _stream_handle(q)))
    return dq, dk, dv


def sdpa_packed_bwd_kernel_name(q, k, v, seq_offsets, **kw) -> str:
    """Which backward kernels mfx_sdpa_packed_bwd picks (host-only query)."""
    torch = _torch()
    lse = torch.empty(q.shape[1], q.shape[0])
    name = load().mfx_sdpa_packed_bwd_kernel_name(
        ctypes.byref(sdpa_packed_bwd_args(q, k, v, q, q, lse, q, k, v, seq_offsets, **kw)))
    if name is None:
        raise MfxError(-1, load().mfx_last_error().decode())
    return name.decode()


# ---- query / key norm with rotation ----------------------------------------------

def rope_table(rot: int, theta: float = 10000.0, *, inv_freq=None, device="cuda"):
    """The frequencies of a rotation of `rot` features, as qk_norm_rope takes
    them: theta^(-2 i / rot) radians per position, or the given inv_freq
    [rot / 2] (scaled frequencies), as 64-bit fractions of a turn
    (mfx_rope_freqs).  Made once and kept, like a weight."""
    torch = _torch()
    out = torch.empty(rot // 2, dtype=torch.int64)
    f = None
    if inv_freq is not None:
        f = torch.as_tensor(inv_freq, dtype=torch.float64).cpu().contiguous()
        if f.shape != (rot // 2,):
            raise ValueError(f"inv_freq must have rot / 2 = {rot // 2} entries")
    check(load().mfx_rope_freqs(float(theta), rot, _ptr(f), out.data_ptr()))
    return out.to(device)


_QK_PACK = struct.Struct("8P6q16q3q4i4ifi").pack
_QK_BWD_PACK = struct.Struct("13PN6q24q3q4i4ifi").pack


def _head_strides(t, layout):
    """(batch, head, seq, feature) strides of [T, H, D] tokens or a 4-D tensor."""
    s = t.stride()
    if len(s) == 3:
        return (0, s[1], s[0], s[2])
    return s if layout == "bhtd" else (s[0], s[2], s[1], s[3])


_NO_ROWS = (0, 0, 0, 1)


def _same(given, like):
    """A caller's output or gradient (or None) against the tensor it belongs to."""
    if (given is None) != (like is None):
        raise ValueError("q and k each need their outputs (and gradients)")
    if given is not None and (given.shape != like.shape or given.dtype != like.dtype):
        raise ValueError("outputs and gradients must have q's and k's shape and dtype")
    return given


def _qk_fields(q, k, positions, table, q_weight, k_weight, eps, sections, interleaved, layout, more):
    """Checked (pointers of positions and table, dims, the rest) for the packed
    structs; the rest starts with the strides of q, k and of the tensors in
    `more` (shaped like q and k in turn)."""
    first = q if q is not None else k
    if first is None:
        raise ValueError("q or k is needed")
    shape = first.shape
    if len(shape) == 3:
        T, H, D = shape
        B, at = 1, 1
    elif len(shape) != 4:
        raise ValueError("queries and keys are [T, H, D] or 4-D")
    elif layout == "bhtd":
        B, H, T, D = shape
        at = 1
    elif layout == "bthd":
        B, T, H, D = shape
        at = 2
    else:
        raise ValueError(f"layout must be 'bhtd' or 'bthd', got {layout!r}")
    code = dtype_code(first.dtype)
    if q is None:
        Hq, Hkv = 0, H
    elif k is None:
        Hq, Hkv = H, 0
    else:
        ks = k.shape
        Hq, Hkv = H, ks[at] if len(ks) == len(shape) else 0
        if k.dtype != first.dtype or (*shape[:at], Hkv, *shape[at + 1:]) != ks:
            raise ValueError("q and k must agree in dtype, batch, tokens and head size")
    strides = ()
    for t in (q, k, *more):
        strides += _NO_ROWS if t is None else _head_strides(t, layout)
    pp = tp = rot = 0
    ps, axes, secs = (0, 0, 0), 1, (0, 0, 0, 0)
    if table is not None:
        torch = _torch()
        rot = 2 * table.shape[0]
        if table.dtype != torch.int64 or table.dim() != 1 or not table.is_contiguous():
            raise ValueError("table must come from rope_table")
        if positions is None or positions.dtype != torch.int32:
            raise TypeError("positions must be an int32 tensor")
        pshape, ps = positions.shape, positions.stride()
        if sections is None:
            secs, ps = (rot // 2, 0, 0, 0), (0, *ps)
        else:
            axes = len(sections)
            if not 1 <= axes <= 4 or len(pshape) < 2 or pshape[0] != axes:
                raise ValueError("positions with sections must be [axes, T] or [axes, B, T], 1 to 4 axes")
            secs, pshape = (*sections, 0, 0, 0)[:4], pshape[1:]
        if len(pshape) == 1 and pshape[0] == T:
            ps = (ps[0], 0, ps[1])
        elif len(pshape) != 2 or pshape[0] != B or pshape[1] != T:
            raise ValueError(f"positions {tuple(positions.shape)} do not fit {B} x {T} tokens")
        pp, tp = positions.data_ptr(), table.data_ptr()
    pd = None
    for w in (q_weight, k_weight):
        if w is not None:
            if w.shape != (D,) or not w.is_contiguous() or (pd is not None and w.dtype != pd):
                raise ValueError("weights must be contiguous [head size] vectors of one dtype")
            pd = w.dtype
    return (pp, tp), (B, T, Hq, Hkv, D, rot), (*strides, *ps, *secs, axes, 1 if interleaved else 0, code,
                                               code if pd is None else dtype_code(pd),
                                               -1.0 if eps is None else _f32(eps), 0)


def qk_norm_rope(q, k, positions, table, *, q_weight=None, k_weight=None, eps=1e-6, sections=None, interleaved=False,
                 layout="bhtd", q_out=None, k_out=None):
    """(q_out, k_out): each head row of q and k normalised by its root mean
    square (times its weight) and turned by its token's position
    (mfx_qk_norm_rope).

    q [T, Hq, D] and k [T, Hkv, D], or 4-D in `layout` ("bhtd" / "bthd"); k (or
    q) may be None.  positions: int32 [T] or [B, T]; with `sections` (pairs per
    position axis) [axes, T] or [axes, B, T].  table: rope_table(rot, ...)
    (None: no rotation, positions unused).  eps None: no norm.  interleaved:
    pairs side by side instead of half the rotated features apart.  The
    outputs are contiguous unless given (q_out may be q, k_out k)."""
    first = q if q is not None else k
    q_out = _fresh(q) if q_out is None else _same(q_out, q)
    k_out = _fresh(k) if k_out is None else _same(k_out, k)
    ptrs, dims, rest = _qk_fields(q, k, positions, table, q_weight, k_weight, eps, sections, interleaved, layout,
                                  (q_out, k_out))
    a = QkNormRopeArgs.from_buffer_copy(_QK_PACK(_ptr(q), _ptr(k), _ptr(q_out), _ptr(k_out), _ptr(q_weight),
                                                 _ptr(k_weight), *ptrs, *dims, *rest))
    with _on(first, q, k, q_out, k_out, q_weight, k_weight, positions, table):
        check(load().mfx_qk_norm_rope(ctypes.byref(a), _stream_handle(first)))
    return q_out, k_out


def qk_norm_rope_bwd(q, k, dq_out, dk_out, positions, table, *, q_weight=None, k_weight=None, eps=1e-6, sections=None,
                     interleaved=False, layout="bhtd", dq=None, dk=None, workspace=None):
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rope for the gradients dq_out,
    dk_out of its outputs (mfx_qk_norm_rope_bwd); q, k are the forward's inputs.
    A weight's gradient has its dtype; None for an absent weight."""
    torch = _torch()
    first = q if q is not None else k
    dq = _fresh(q) if dq is None else _same(dq, q)
    dk = _fresh(k) if dk is None else _same(dk, k)
    ptrs, dims, rest = _qk_fields(q, k, positions, table, q_weight, k_weight, eps, sections, interleaved, layout,
                                  (_same(dq_out, q), _same(dk_out, k), dq, dk))
    dqw = torch.empty_like(q_weight) if q_weight is not None else None
    dkw = torch.empty_like(k_weight) if k_weight is not None else None
    a = QkNormRopeBwdArgs.from_buffer_copy(_QK_BWD_PACK(
        _ptr(q), _ptr(k), _ptr(dq_out), _ptr(dk_out), _ptr(dq), _ptr(dk), _ptr(q_weight), _ptr(k_weight), _ptr(dqw),
        _ptr(dkw), *ptrs, 0, 0, *dims, *rest))
    with _on(first, q, k, dq_out, dk_out, dq, dk, q_weight, k_weight, positions, table, workspace):
        keep = _workspace(a, "mfx_qk_norm_rope_bwd_workspace_size", workspace, first)  # noqa: F841 (until the launch)
        check(load().mfx_qk_norm_rope_bwd(ctypes.byref(a), _stream_handle(first)))
    return dq, dk, dqw, dkw


# ---- cross entropy of a linear head ----------------------------------------------

_XENT_PACK = struct.Struct("6PN5q2i").pack
_XENT_BWD_PACK = struct.Struct("8PN7q4i").pack


def _xent_dims(h, w, targets):
    """((T, H, V), h_stride, w_stride, dtype, target dtype) of checked tensors."""
    torch = _torch()
    if w.dim() != 2 or h.dim() < 2 or w.shape[1] != h.shape[-1]:
        raise ValueError("h is [..., H] and w [V, H]")
    if w.dtype != h.dtype:
        raise ValueError("h and w must share one dtype")
    if targets.shape != h.shape[:-1] or not targets.is_contiguous():
        raise ValueError("targets must be contiguous, one for each row of h")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("targets must be int32 or int64")
    if w.stride(1) != 1:
        raise ValueError("last dimension must be contiguous")
    T, H, hs = _rows_view(h)
    # (One row may carry any stride.)
    return ((T, H, w.shape[0]), hs if T > 1 else H, w.stride(0) if w.shape[0] > 1 else H, dtype_code(h.dtype),
            MFX_I64 if targets.dtype == torch.int64 else MFX_I32)


def _f32_rows(name, t, like):
    if t.dtype != _torch().float32 or t.shape != like.shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous f32 tensor of the targets' shape")


def linear_xent(h, w, targets, *, loss=None, lse=None, workspace=None):
    """(loss, lse) of softmax cross entropy with logits h w^T, which are never
    stored (mfx_linear_xent): h [..., H], w [V, H], targets [...] int32 or
    int64.  A target outside [0, V) marks a row that does not count (loss 0).
    loss and lse are f32 of the targets' shape."""
    torch = _torch()
    dims, hs, ws, code, tcode = _xent_dims(h, w, targets)
    if loss is None:
        loss = torch.empty(targets.shape, dtype=torch.float32, device=h.device)
    if lse is None:
        lse = torch.empty(targets.shape, dtype=torch.float32, device=h.device)
    _f32_rows("loss", loss, targets)
    _f32_rows("lse", lse, targets)
    a = LinearXentArgs.from_buffer_copy(_XENT_PACK(h.data_ptr(), w.data_ptr(), targets.data_ptr(), loss.data_ptr(),
                                                   lse.data_ptr(), 0, 0, *dims, hs, ws, code, tcode))
    with _on(h, w, targets, loss, lse, workspace):
        keep = _workspace(a, "mfx_linear_xent_workspace_size", workspace, h)  # noqa: F841 (until the launch)
        check(load().mfx_linear_xent(ctypes.byref(a), _stream_handle(h)))
    return loss, lse


def linear_xent_bwd(h, w, targets, lse, dloss, *, need_dh=True, need_dw=True, dw_dtype=None, dh=None, dw=None,
                    workspace=None):
    """(dh, dw) of linear_xent for the gradients dloss of its losses, from its
    lse (mfx_linear_xent_bwd).  dw has w's dtype or `dw_dtype` (f32); one not
    needed is None and costs nothing."""
    torch = _torch()
    dims, hs, ws, code, tcode = _xent_dims(h, w, targets)
    _f32_rows("lse", lse, targets)
    _f32_rows("dloss", dloss, targets)
    if dh is None and need_dh:
        dh = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    if dw is None and need_dw:
        dw = torch.empty(w.shape, dtype=dw_dtype or w.dtype, device=w.device)
    if dh is not None and (dh.shape != h.shape or dh.dtype != h.dtype):
        raise ValueError("dh must match h")
    if dw is not None and (dw.shape != w.shape or dw.stride(1) != 1):
        raise ValueError("dw must match w")
    dhs = _rows_view(dh)[2] if dh is not None and dims[0] > 1 else dims[1]
    dws = dw.stride(0) if dw is not None and dims[2] > 1 else dims[1]
    a = LinearXentBwdArgs.from_buffer_copy(_XENT_BWD_PACK(
        h.data_ptr(), w.data_ptr(), targets.data_ptr(), lse.data_ptr(), dloss.data_ptr(), _ptr(dh), _ptr(dw), 0, 0,
        *dims, hs, ws, dhs, dws, code, tcode, dtype_code(dw.dtype) if dw is not None else code, 0))
    with _on(h, w, targets, lse, dloss, dh, dw, workspace):
        keep = _workspace(a, "mfx_linear_xent_bwd_workspace_size", workspace, h)  # noqa: F841 (until the launch)
        check(load().mfx_linear_xent_bwd(ctypes.byref(a), _stream_handle(h)))
    return dh, dw


# ---- GEMM ----------------------------------------------------------------------

def _matrix(x):
    """(batch, rows, cols, ld, batch_stride) of a 2-D or 3-D tensor whose
    last dim is contiguous."""
    if x.dim() not in (2, 3) or x.stride(-1) != 1:
        raise ValueError("GEMM operands are 2-D or 3-D with a contiguous last dim")
    if x.dim() == 2:
        return 1, x.shape[0], x.shape[1], x.stride(0), 0
    return x.shape[0], x.shape[1], x.shape[2], x.stride(1), x.stride(0)


def gemm_args(a, b, c=None, trans_a=False, trans_b=False):
    """GemmArgs for c = op(a) @ op(b) (row-major, optionally batched; b may
    be 2-D and shared by every batch of a).  trans_a: a is stored [k, m];
    trans_b: b is stored [n, k]."""
    ba, r, s_, lda, sa = _matrix(a)
    m, k = (s_, r) if trans_a else (r, s_)
    bb, r2, s2, ldb, sb = _matrix(b)
    k2, n = (s2, r2) if trans_b else (r2, s2)
    if k2 != k or (bb != ba and bb != 1):
        raise ValueError("GEMM extents disagree")
    return GemmArgs(a.data_ptr(), b.data_ptr(), c.data_ptr() if c is not None else None, dtype_code(a.dtype),
                    dtype_code(c.dtype) if c is not None else MFX_F32, ba, m, n, k, lda, ldb, n, sa,
                    sb if bb > 1 else 0, m * n, int(trans_a), int(trans_b))


def gemm(a, b, out=None, trans_a=False, trans_b=False, out_dtype=None):
    """mfx_gemm: op(a) [(batch,) m, k] @ op(b) [(batch,) k, n] into a new
    contiguous tensor of out_dtype (default f32), or `out`.  trans_a: a is
    stored [(batch,) k, m]; trans_b: b is stored [(batch,) n, k]."""
    torch = _torch()
    _require_gpu(a, b)
    batch = a.shape[0] if a.dim() == 3 else None
    m = a.shape[-1] if trans_a else a.shape[-2]
    n = b.shape[-2] if trans_b else b.shape[-1]
    shape = (batch, m, n) if batch is not None else (m, n)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or torch.float32, device=a.device)
    g = gemm_args(a, b, out, trans_a, trans_b)
    check(load().mfx_gemm(ctypes.byref(g), _stream_handle(a)))
    return out


def gemm_kernel_name(a, b, out=None, trans_a=False, trans_b=False) -> str:
    """Kernel mfx_gemm runs for op(a) @ op(b): "gemm_f32_tile",
    "gemm_bf16_tile", "gemm_f16_tile" or "rocblas"."""
    return load().mfx_gemm_kernel_name(ctypes.byref(gemm_args(a, b, out, trans_a, trans_b))).decode()


def _bind_inputs(prog, tensors):
    keep = []
    for i, t in enumerate(tensors):
        prog.inputs[i].data = t.data_ptr() if t is not None else None
        keep.append(t)
    return keep


def gemm_ew(a, b, prog, c_input, inputs, out):
    """mfx_gemm_ew: out = prog(inputs) with inputs[c_input] the product a @ b
    (pass None for it)."""
    _require_gpu(a, b, out)
    g = gemm_args(a, b)
    prog.out = out.data_ptr()
    _bind_inputs(prog, inputs)
    check(load().mfx_gemm_ew(ctypes.byref(g), ctypes.byref(prog), c_input, _stream_handle(a)))
    return out


def elementwise(prog, inputs, out):
    """mfx_elementwise: out = prog(inputs)."""
    _require_gpu(out)
    prog.out = out.data_ptr()
    _bind_inputs(prog, inputs)
    check(load().mfx_elementwise(ctypes.byref(prog), _stream_handle(out)))
    return out


def gemm_ew_source(g, prog, c_input) -> str | None:
    """Generated source of the fused kernel (None when the pair is not fused)."""
    lib = load()
    n = lib.mfx_gemm_ew_source(ctypes.byref(g), ctypes.byref(prog), c_input, None, 0)
    if n < 0:
        return None
    buf = ctypes.create_string_buffer(int(n) + 1)
    lib.mfx_gemm_ew_source(ctypes.byref(g), ctypes.byref(prog), c_input, buf, n + 1)
    return buf.value.decode()
