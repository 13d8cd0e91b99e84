"""ctypes binding of libtsa.so, the C-ABI declared in include/tsa.h, for torch tensors.

torch is only plumbing here (device memory and the current HIP stream); every call goes
straight to the hand-written gfx950 kernels.  There is no fallback: if the library is
missing or a call fails, an exception is raised.

Shapes and dtypes mirror the reference labs (cookys/turing-sm75):
  attention  q, k, v, o      [B, H, S, D] fp16                (src/attn_sm75.cu:64,254)
  GDN        q, k            [B, T, Hq, dk] fp16              (src/gdn_sm75.cu:75-77)
             v, out          [B, T, Hv, dv] fp16
             g_log, beta     [B, T, Hv] fp32
             state           [B, Hv, dv, dk] fp32, updated in place (:71-72,1094)
  decode     q, k [B, Hq, dk], v/out [B, Hv, dv], g_log/beta [B, Hv]
"""
from __future__ import annotations

import ctypes
import math
import os
import re
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(_HERE)
LIB_PATH = os.path.join(PKG_ROOT, "lib", "libtsa.so")
HEADER_PATH = os.path.join(os.path.dirname(PKG_ROOT), "include", "tsa.h")

TSA_OK = 0
TSA_ERR_NULL = 1
TSA_ERR_SHAPE = 2
TSA_ERR_UNSUPPORTED = 3
TSA_ERR_WORKSPACE = 4
TSA_ERR_LAUNCH = 5
TSA_ERR_ARG = 6
TSA_ERR_SCRATCH = 7

TSA_TYPE_F32, TSA_TYPE_F16 = 0, 1


class TsaTensor(ctypes.Structure):
    """The tsa_tensor view of include/tsa.h (the fields of a ggml_tensor view)."""
    _fields_ = [("data", ctypes.c_void_p), ("type", ctypes.c_int),
                ("ne", ctypes.c_int64 * 4), ("nb", ctypes.c_size_t * 4)]


class TsaKv8(ctypes.Structure):
    """The tsa_kv8 cache of include/tsa.h."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "k_sum", "k_sum_scale", "k_open",
                                               "v_open", "table")] + \
               [(n, ctypes.c_int) for n in ("B", "Hkv", "D", "n_pages", "max_blocks")]


class TsaRows(ctypes.Structure):
    """The tsa_rows view of include/tsa.h."""
    _fields_ = [("data", ctypes.c_void_p), ("stride_b", ctypes.c_int64), ("stride_h", ctypes.c_int64),
                ("stride_t", ctypes.c_int64)]


class TsaRopeParams(ctypes.Structure):
    """The tsa_rope_params of include/tsa.h."""
    _fields_ = [(n, ctypes.c_double) for n in ("base", "factor", "beta_fast", "beta_slow", "low", "high")] + \
               [(n, ctypes.c_int) for n in ("rot", "scaling", "orig_len")]


class TsaRopePlan(ctypes.Structure):
    """The tsa_rope_plan of include/tsa.h."""
    _fields_ = [("freq", ctypes.c_void_p), ("amp", ctypes.c_float), ("rot", ctypes.c_int), ("interleaved", ctypes.c_int)]


_tp = ctypes.POINTER(TsaTensor)


_vp, _i, _f, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
_SIGNATURES = {
    "tsa_strerror": (ctypes.c_char_p, [_i]),
    "tsa_version": (ctypes.c_char_p, []),
    "tsa_attn_fwd": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _i, _vp]),
    "tsa_attn_naive": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _i, _vp]),
    "tsa_attn_fwd_valu": (_i, [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _i, _vp]),
    "tsa_attn_gqa_fwd": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _i, _vp]),
    "tsa_attn_gqa_naive": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _i, _vp]),
    "tsa_gdn_chunked_workspace_bytes": (_sz, [_i] * 7),
    "tsa_gdn_chunked_fwd": (_i, [_vp] * 7 + [_i] * 7 + [_f, _vp, _sz, _vp]),
    "tsa_gdn_chunked_fwd_noalloc": (_i, [_vp] * 7 + [_i] * 7 + [_f, _vp]),
    "tsa_gdn_chunked_redo_count": (_i, [_vp, _sz] + [_i] * 8 + [ctypes.POINTER(ctypes.c_int), _vp]),
    "tsa_gdn_chunked_workspace_bytes_f32": (_sz, [_i] * 7),
    "tsa_gdn_chunked_plan_workspace_bytes": (_sz, [_i] * 9),
    "tsa_gdn_chunked_plan_fwd": (_i, [_vp] * 7 + [_i] * 7 + [_f, _i, _i, _vp, _sz, _vp]),
    "tsa_gdn_chunked_fwd_f32": (_i, [_vp] * 7 + [_i] * 7 + [_f, _vp, _sz, _vp]),
    "tsa_gdn_recurrent_fwd_f32": (_i, [_vp] * 7 + [_i] * 6 + [_f, _vp]),
    "tsa_gdn_decode_step_f32": (_i, [_vp] * 7 + [_i] * 5 + [_f, _vp]),
    "tsa_gdn_naive_f32": (_i, [_vp] * 7 + [_i] * 6 + [_f, _vp]),
    "tsa_gdn_recurrent_fwd": (_i, [_vp] * 7 + [_i] * 6 + [_f, _vp]),
    "tsa_gdn_decode_step": (_i, [_vp] * 7 + [_i] * 5 + [_f, _vp]),
    "tsa_gdn_naive": (_i, [_vp] * 7 + [_i] * 6 + [_f, _vp]),
    "tsa_gdn_chunked_fused_fwd": (_i, [_vp] * 9 + [_i] * 7 + [_f, _f, _vp, _sz, _vp]),
    "tsa_gdn_decode_fused_step": (_i, [_vp] * 9 + [_i] * 5 + [_f, _f, _vp]),
    "tsa_gdn_preprocess": (_i, [_vp] * 10 + [_i] * 5 + [_f, _vp]),
    "tsa_gdn_gated_rmsnorm": (_i, [_vp] * 4 + [_i] * 4 + [_f, _vp]),
    "tsa_ggml_gdn_workspace_bytes": (_sz, [_tp, _tp]),
    "tsa_ggml_gated_delta_net": (_i, [_tp] * 8 + [_f, _vp, _sz, _vp]),
    "tsa_kv8_write": (_i, [_vp] * 5 + [_i, _vp]),
    "tsa_kv8_read": (_i, [_vp] * 3 + [_i] + [_vp] * 3),
    "tsa_kv8_workspace_bytes": (_sz, [_vp] + [_i] * 4),
    "tsa_attn_kv8_fwd": (_i, [_vp] * 6 + [_i] * 3 + [_f, _i, _vp, _sz, _vp]),
    "tsa_kv8_select": (_i, [_vp] * 4 + [_i] * 5 + [_vp, _i, _vp, _sz, _vp]),
    "tsa_rope_freqs": (_i, [_vp] * 3),
    "tsa_rope": (_i, [_vp, _i, _vp, _vp, _i, _vp, _vp, _i] + [_vp] * 3 + [_i] * 4 + [_vp]),
    "tsa_attn_train_fwd": (_i, [_vp] * 8 + [_i] * 6 + [_f, _i, _vp]),
    "tsa_attn_bwd_workspace_bytes": (_sz, [_i] * 8),
    "tsa_attn_bwd": (_i, [_vp] * 13 + [_i] * 6 + [_f, _i, _vp, _sz, _vp]),
    "tsa_attn_kv8_blocks_fwd": (_i, [_vp] * 6 + [_i] * 2 + [_vp, _i, _f, _vp, _sz, _vp]),
}


class TsaError(RuntimeError):
    """A tsa_* entry point returned a non-zero code."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"tsa error {code}: {msg}")
        self.code = code


_lib = None


def load(path: str | None = None) -> ctypes.CDLL:
    """Load libtsa.so once (raises OSError with a build hint when it is missing).  The
    environment variable TSA_LIB_PATH names another build of the same library (the tests'
    sanitizer run uses it)."""
    global _lib
    if _lib is None:
        path = path or os.environ.get("TSA_LIB_PATH") or LIB_PATH
        if not os.path.exists(path):
            raise OSError(f"{path} not found: build it with `make -C turing-sm75_amd` "
                          "(or __graft_entry__.build())")
        lib = ctypes.CDLL(path)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def header_symbols(path: str = HEADER_PATH) -> list[str]:
    """Names of the functions include/tsa.h declares."""
    text = open(path).read()
    return sorted(set(re.findall(r"\b(tsa_[a-z0-9_]+)\s*\(", text)))


def strerror(code: int) -> str:
    return load().tsa_strerror(code).decode()


def _check(code: int) -> None:
    if code != TSA_OK:
        raise TsaError(code, strerror(code))


# What every call does on the host is longer than a small call's kernel (a decode step of one
# sequence: 4 us on the GPU), so the checks and conversions below avoid what only costs time:
# no Stream object for the current stream, pointers as plain ints (ctypes converts them by the
# declared argument types), torch looked up once, a workspace sized only when one is made.
_torch = None


def _t():
    global _torch
    if _torch is None:
        import torch
        _torch = torch
    return _torch


def _stream(stream):
    if stream is None:
        torch = _torch or _t()
        if not torch.cuda.is_initialized():
            return torch.cuda.current_stream().cuda_stream
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    return stream.cuda_stream


def _need(t, dtype, ndim, name):
    if not isinstance(t, (_torch or _t()).Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype or t.dim() != ndim or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {ndim}-d {dtype} CUDA tensor, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _ptr(t):
    return t.data_ptr()


def _out(out, like, name="out"):
    """The output tensor: a new one shaped like `like`, or the caller's, which must have
    exactly that shape (a smaller one would be written past its end)."""
    if out is None:
        return (_torch or _t()).empty_like(like)
    _need(out, like.dtype, like.dim(), name)
    if out.shape != like.shape:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)}, got {tuple(out.shape)}")
    return out


def _scratch(nbytes, device, stream):
    """A workspace for one call.  It is allocated on the stream the kernels run on, so the
    caching allocator does not hand it out again before they have finished with it."""
    import torch
    s = torch.cuda.current_stream(device) if stream is None else stream
    with torch.cuda.stream(s):
        return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
def attn_fwd(q, k, v, out=None, scale=None, causal=True, stream=None, naive=False, valu=False):
    """O = softmax(scale Q K^T [+ causal mask]) V on the MFMA kernel (or the naive one, or the
    VALU opponent with valu=True)."""
    torch = _torch or _t()
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t, torch.float16, 4, name)
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q, k, v shapes differ: {tuple(q.shape)} {tuple(k.shape)} {tuple(v.shape)}")
    B, H, S, D = q.shape
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.float16, 4, "out")
    if out.shape != q.shape:
        raise ValueError("out shape differs from q")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if naive and valu:
        raise ValueError("naive and valu select different kernels")
    fn = load().tsa_attn_naive if naive else (load().tsa_attn_fwd_valu if valu else load().tsa_attn_fwd)
    _check(fn(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, H, S, D, float(scale), int(bool(causal)),
              _stream(stream)))
    return out


def attn_gqa_fwd(q, k, v, gate=None, out=None, scale=None, causal=True, stream=None, naive=False):
    """Gated grouped-query attention: q, gate [B, Hq, S, D]; k, v [B, Hkv, S, D] with
    Hq % Hkv == 0; O = softmax(scale Q K^T [+ causal mask]) V, times sigmoid(gate) if given."""
    torch = _torch or _t()
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t, torch.float16, 4, name)
    B, Hq, S, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (B, Hkv, S, D) or v.shape != k.shape:
        raise ValueError(f"k, v must be [B, Hkv, S, D] with q's B, S, D: {tuple(q.shape)} "
                         f"{tuple(k.shape)} {tuple(v.shape)}")
    if gate is not None:
        _need(gate, torch.float16, 4, "gate")
        if gate.shape != q.shape:
            raise ValueError("gate shape differs from q")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.float16, 4, "out")
    if out.shape != q.shape:
        raise ValueError("out shape differs from q")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    fn = load().tsa_attn_gqa_naive if naive else load().tsa_attn_gqa_fwd
    gp = _ptr(gate) if gate is not None else None
    _check(fn(_ptr(q), _ptr(k), _ptr(v), gp, _ptr(out), B, Hq, Hkv, S, D, float(scale),
              int(bool(causal)), _stream(stream)))
    return out


# ---------------------------------------------------------------------------------------
# Gated DeltaNet
# ---------------------------------------------------------------------------------------
def _gdn_shapes(q, k, v, g_log, beta, state, batched_t: bool):
    """Shapes of a GDN call; q, k, v are all fp16 (the library's I/O type) or all fp32 (the
    *_f32 entry points, the reference's own I/O)."""
    torch = _torch or _t()
    nd = 4 if batched_t else 3
    io = q.dtype if isinstance(q, torch.Tensor) and q.dtype in (torch.float16, torch.float32) else torch.float16
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t, io, nd, name)
    _need(g_log, torch.float32, nd - 1, "g_log")
    _need(beta, torch.float32, nd - 1, "beta")
    _need(state, torch.float32, 4, "state")
    if batched_t:
        B, T, Hq, dk = q.shape
        Hv, dv = v.shape[2], v.shape[3]
        ok = (k.shape == q.shape and v.shape[:2] == (B, T) and g_log.shape == (B, T, Hv)
              and beta.shape == (B, T, Hv) and state.shape == (B, Hv, dv, dk))
    else:
        B, Hq, dk = q.shape
        Hv, dv = v.shape[1], v.shape[2]
        T = 1
        ok = (k.shape == q.shape and v.shape[0] == B and g_log.shape == (B, Hv)
              and beta.shape == (B, Hv) and state.shape == (B, Hv, dv, dk))
    if not ok:
        raise ValueError("inconsistent GDN shapes: q %s k %s v %s g %s beta %s state %s" % (
            tuple(q.shape), tuple(k.shape), tuple(v.shape), tuple(g_log.shape),
            tuple(beta.shape), tuple(state.shape)))
    return B, T, Hq, Hv, dk, dv


def gdn_chunked_workspace_bytes(B, T, Hq, Hv, dk=128, dv=128, chunk=64, f32=False, nseg=None) -> int:
    """Workspace bytes of one chunked call.  With few heads and many chunks the library's plan
    splits the sequence and needs more; the plan is a function of the shapes.  nseg asks for
    an explicit plan (0 = the library's, 1 = no split, n >= 2 = n segments)."""
    if nseg is not None:
        return int(load().tsa_gdn_chunked_plan_workspace_bytes(B, T, Hq, Hv, dk, dv, chunk, int(bool(f32)),
                                                               int(nseg)))
    fn = load().tsa_gdn_chunked_workspace_bytes_f32 if f32 else load().tsa_gdn_chunked_workspace_bytes
    return int(fn(B, T, Hq, Hv, dk, dv, chunk))


def gdn_chunked_fwd(q, k, v, g_log, beta, state, out=None, scale=None, chunk=64, ws=None,
                    stream=None, nseg=None):
    """Chunked prefill; state [B, Hv, dv, dk] is updated in place; returns out.  fp32 q/k/v
    select tsa_gdn_chunked_fwd_f32 (fp32 out).  With few heads (B*Hv <= 21) and at least 16
    chunks the library splits the sequence into segments run side by side (same results to
    fp32 rounding).  nseg (through tsa_gdn_chunked_plan_fwd) asks for an explicit plan: 0 =
    the library's, 1 = no split, n >= 2 = n segments."""
    torch = _torch or _t()
    B, T, Hq, Hv, dk, dv = _gdn_shapes(q, k, v, g_log, beta, state, True)
    out = _out(out, v)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    f32 = q.dtype == torch.float32
    if ws is None:
        ws = _scratch(gdn_chunked_workspace_bytes(B, T, Hq, Hv, dk, dv, chunk, f32=f32, nseg=nseg), q.device, stream)
    args = (_ptr(q), _ptr(k), _ptr(v), _ptr(g_log), _ptr(beta), _ptr(state), _ptr(out),
            B, T, Hq, Hv, dk, dv, chunk, float(scale))
    tail = (_ptr(ws), ws.numel() * ws.element_size(), _stream(stream))
    if nseg is not None:
        _check(load().tsa_gdn_chunked_plan_fwd(*args, int(f32), int(nseg), *tail))
    else:
        fn = load().tsa_gdn_chunked_fwd_f32 if f32 else load().tsa_gdn_chunked_fwd
        _check(fn(*args, *tail))
    return out


def gdn_chunked_redo_count(ws, B, T, Hq, Hv, dk=128, dv=128, chunk=64, f32=False, stream=None) -> int:
    """Carry workgroups of the last chunked call on ws that were redone after a timed-out wait
    (0 when prep and carry ran side by side); synchronises the stream."""
    c = ctypes.c_int(-1)
    _check(load().tsa_gdn_chunked_redo_count(_ptr(ws), ws.numel() * ws.element_size(), B, T, Hq,
                                             Hv, dk, dv, chunk, int(bool(f32)), ctypes.byref(c),
                                             _stream(stream)))
    return c.value


def gdn_recurrent_fwd(q, k, v, g_log, beta, state, out=None, scale=None, stream=None,
                      naive=False):
    """Token-serial recurrence over T tokens (or the naive check kernel); state in place.
    fp32 q/k/v select the *_f32 entry points."""
    torch = _torch or _t()
    B, T, Hq, Hv, dk, dv = _gdn_shapes(q, k, v, g_log, beta, state, True)
    out = _out(out, v)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    sfx = "_f32" if q.dtype == torch.float32 else ""
    fn = getattr(load(), ("tsa_gdn_naive" if naive else "tsa_gdn_recurrent_fwd") + sfx)
    _check(fn(_ptr(q), _ptr(k), _ptr(v), _ptr(g_log), _ptr(beta), _ptr(state), _ptr(out),
              B, T, Hq, Hv, dk, dv, float(scale), _stream(stream)))
    return out


def gdn_decode_step(q, k, v, g_log, beta, state, out=None, scale=None, stream=None):
    """One token per sequence: q/k [B, Hq, dk], v [B, Hv, dv]; state in place (fp16 or fp32
    q/k/v/out)."""
    torch = _torch or _t()
    B, _, Hq, Hv, dk, dv = _gdn_shapes(q, k, v, g_log, beta, state, False)
    out = _out(out, v)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    fn = load().tsa_gdn_decode_step_f32 if q.dtype == torch.float32 else load().tsa_gdn_decode_step
    _check(fn(
        _ptr(q), _ptr(k), _ptr(v), _ptr(g_log), _ptr(beta), _ptr(state), _ptr(out),
        B, Hq, Hv, dk, dv, float(scale), _stream(stream)))
    return out


def gdn_naive(q, k, v, g_log, beta, state, out=None, scale=None, stream=None):
    """The naive on-device check kernel (one thread per state column)."""
    return gdn_recurrent_fwd(q, k, v, g_log, beta, state, out, scale, stream, naive=True)


# ---- the layer's pre / post ops (q, k l2 norm; beta = sigmoid(b); g_log = softplus(a +
# dt_bias) * A; gated RMSNorm of the output), fused or as passes of their own ----
def _gates(a, b, dt_bias, A, lead, Hv):
    torch = _torch or _t()
    for name, t in (("a", a), ("b", b)):
        _need(t, torch.float32, len(lead) + 1, name)
        if tuple(t.shape) != tuple(lead) + (Hv,):
            raise ValueError(f"{name}: expected shape {tuple(lead) + (Hv,)}, got {tuple(t.shape)}")
    for name, t in (("dt_bias", dt_bias), ("A", A)):
        _need(t, torch.float32, 1, name)
        if t.numel() != Hv:
            raise ValueError(f"{name}: expected {Hv} values, got {t.numel()}")


def gdn_chunked_fused_fwd(q, k, v, a, b, dt_bias, A, state, out=None, scale=None, eps=1e-6,
                          chunk=64, ws=None, stream=None):
    """Chunked prefill from raw q, k [B,T,Hq,dk] and raw gate projections a, b [B,T,Hv]
    (fp16 q / k / v / out)."""
    torch = _torch or _t()
    _need(q, torch.float16, 4, "q")
    B, T, Hq, Hv, dk, dv = _gdn_shapes(q, k, v, a, b, state, True)
    _gates(a, b, dt_bias, A, (B, T), Hv)
    out = _out(out, v)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    if ws is None:
        ws = _scratch(gdn_chunked_workspace_bytes(B, T, Hq, Hv, dk, dv, chunk), q.device, stream)
    _check(load().tsa_gdn_chunked_fused_fwd(
        _ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b), _ptr(dt_bias), _ptr(A), _ptr(state),
        _ptr(out), B, T, Hq, Hv, dk, dv, chunk, float(scale), float(eps), _ptr(ws),
        ws.numel() * ws.element_size(), _stream(stream)))
    return out


def gdn_decode_fused_step(q, k, v, a, b, dt_bias, A, state, out=None, scale=None, eps=1e-6,
                          stream=None):
    """One decode step from raw q, k [B,Hq,dk] and raw gate projections a, b [B,Hv] (fp16
    q / k / v / out)."""
    torch = _torch or _t()
    _need(q, torch.float16, 3, "q")
    B, _, Hq, Hv, dk, dv = _gdn_shapes(q, k, v, a, b, state, False)
    _gates(a, b, dt_bias, A, (B,), Hv)
    out = _out(out, v)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    _check(load().tsa_gdn_decode_fused_step(
        _ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b), _ptr(dt_bias), _ptr(A), _ptr(state),
        _ptr(out), B, Hq, Hv, dk, dv, float(scale), float(eps), _stream(stream)))
    return out


def gdn_preprocess(q, k, a, b, dt_bias, A, eps=1e-6, stream=None):
    """The pre-ops as a pass: returns (q_n, k_n, g_log, beta) for raw q, k [B,T,Hq,dk]."""
    torch = _torch or _t()
    _need(q, torch.float16, 4, "q")
    _need(k, torch.float16, 4, "k")
    if k.shape != q.shape:
        raise ValueError("q and k must have the same shape")
    B, T, Hq, dk = q.shape
    Hv = a.shape[-1]
    _gates(a, b, dt_bias, A, (B, T), Hv)
    qn, kn = torch.empty_like(q), torch.empty_like(k)
    g_log, beta = torch.empty_like(a), torch.empty_like(b)
    _check(load().tsa_gdn_preprocess(
        _ptr(q), _ptr(k), _ptr(a), _ptr(b), _ptr(dt_bias), _ptr(A), _ptr(qn), _ptr(kn),
        _ptr(g_log), _ptr(beta), B, T, Hq, Hv, dk, float(eps), _stream(stream)))
    return qn, kn, g_log, beta


def gdn_gated_rmsnorm(x, z, w, out=None, eps=1e-6, stream=None):
    """y = x / sqrt(mean(x^2) + eps) * w * silu(z) over dv; x, z [B,T,Hv,dv] fp16, w [dv]."""
    torch = _torch or _t()
    _need(x, torch.float16, 4, "x")
    _need(z, torch.float16, 4, "z")
    _need(w, torch.float32, 1, "w")
    if z.shape != x.shape or w.numel() != x.shape[3]:
        raise ValueError("inconsistent shapes: x %s z %s w %s" % (tuple(x.shape), tuple(z.shape),
                                                                 tuple(w.shape)))
    out = _out(out, x)
    B, T, Hv, dv = x.shape
    _check(load().tsa_gdn_gated_rmsnorm(_ptr(x), _ptr(z), _ptr(w), _ptr(out), B, T, Hv, dv,
                                        float(eps), _stream(stream)))
    return out


# ---- ggml-layout adapter ----
def ggml_view(t) -> TsaTensor:
    """The ggml view of a torch tensor of up to 4 dims: ne / nb are its shape / strides in
    reverse order (ne[0] = the innermost dimension), padded with 1s."""
    torch = _torch or _t()
    return TsaTensor.from_buffer(bytearray(_pack_view(t)))


# a tsa_tensor as bytes: data, type, ne[4], nb[4]
_VIEW = struct.Struct("@Pi4x4q4N")
assert _VIEW.size == ctypes.sizeof(TsaTensor)


def _pack_view(t) -> bytes:
    torch = _torch or _t()
    if t.dtype is torch.float32:
        kind, es = TSA_TYPE_F32, 4
    elif t.dtype is torch.float16:
        kind, es = TSA_TYPE_F16, 2
    else:
        raise ValueError(f"ggml views are fp32 or fp16, got {t.dtype}")
    nd = t.dim()
    if nd > 4 or not t.is_cuda:
        raise ValueError("a ggml view is a CUDA tensor of at most 4 dims")
    ne, nb = list(t.shape[::-1]), [st * es for st in t.stride()[::-1]]
    while len(nb) < 4:
        nb.append(nb[-1] * ne[-1] if nb else es)
        ne.append(1)
    return _VIEW.pack(t.data_ptr(), kind, *ne, *nb)


def ggml_gdn_workspace_bytes(q, v) -> int:
    return int(load().tsa_ggml_gdn_workspace_bytes(ctypes.byref(ggml_view(q)), ctypes.byref(ggml_view(v))))


def ggml_gated_delta_net(q, k, v, g_log, beta, state, out, state_out=None, scale=None, ws=None,
                         stream=None):
    """Torch tensors in the kernels' index order ([B, T, H, S] for q / k / v / out,
    [B, T, Hv] for g_log / beta, [B, Hv, S, S] for the states), any strides / fp32 or fp16:
    passed as ggml views.  state_out defaults to state (in place)."""
    torch = _torch or _t()
    if state_out is None:
        state_out = state
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    if ws is None:
        ws = _scratch(ggml_gdn_workspace_bytes(q, v), q.device, stream)
    views = (TsaTensor * 8).from_buffer(bytearray(b"".join(
        [_pack_view(x) for x in (q, k, v, g_log, beta, state, out, state_out)])))
    _check(load().tsa_ggml_gated_delta_net(*views, float(scale), _ptr(ws), ws.numel() * ws.element_size(),
                                           _stream(stream)))
    return out


# ---------------------------------------------------------------------------------------
# the 8-bit K/V cache and the attention that reads it
# ---------------------------------------------------------------------------------------
KV8_BLOCK = 64


class Kv8Cache:
    """The 8-bit K/V cache of one attention layer for B sequences of at most max_len tokens: codes
    and scales of full blocks of 64 tokens in n_pages pages, the open blocks' rows in fp16
    (include/tsa.h, tsa_kv8).  Without n_pages every sequence has pages of its own for max_len
    tokens; with it, `table` ([B, blocks] int32, -1: no page) is the caller's to fill, in place,
    before a block is written or read."""

    def __init__(self, B, Hkv, D, max_len, n_pages=None, device="cuda"):
        torch = _torch or _t()
        if torch.device(device).type != "cuda":
            raise ValueError(f"a cache lies on a GPU, not on {device}")
        for name, x in (("B", B), ("Hkv", Hkv), ("max_len", max_len)):
            if x < 1:
                raise ValueError(f"{name} must be at least 1, got {x}")
        if D not in (64, 128, 256):
            raise ValueError(f"D must be 64, 128 or 256, got {D}")
        blocks = -(-max_len // KV8_BLOCK)
        own = n_pages is None
        if own:
            n_pages = B * blocks
        if n_pages < 1:
            raise ValueError(f"n_pages must be at least 1, got {n_pages}")
        z = lambda dtype, *shape: torch.zeros(*shape, dtype=dtype, device=device)  # noqa: E731
        self.k, self.v = (z(torch.uint8, n_pages, Hkv, KV8_BLOCK * D) for _ in range(2))
        self.k_scale, self.v_scale, self.k_sum_scale = (z(torch.float32, n_pages, Hkv) for _ in range(3))
        self.k_sum = z(torch.int8, n_pages, Hkv, D)
        self.k_open, self.v_open = (z(torch.float16, B, 2, Hkv, KV8_BLOCK * D) for _ in range(2))
        self.table = torch.arange(n_pages, dtype=torch.int32, device=device).view(B, blocks) if own else \
            torch.full((B, blocks), -1, dtype=torch.int32, device=device)
        self.B, self.Hkv, self.D, self.n_pages, self.max_blocks = B, Hkv, D, n_pages, blocks
        self.max_len = blocks * KV8_BLOCK
        self.device, self.index, self.counts_shape = self.k.device, self.k.get_device(), (B,)
        self.view = TsaKv8(*(_ptr(getattr(self, n)) for n, _ in TsaKv8._fields_[:9]), B, Hkv, D, n_pages, blocks)
        self._ref = ctypes.byref(self.view)


# a tsa_rows as bytes: data, strides of b, h and t.  ctypes passes bytes as a pointer to them, so a
# call's views need no object of their own.
_ROWS = struct.Struct("@P3q")
assert _ROWS.size == ctypes.sizeof(TsaRows)


def _rows(t, shape, name, cache):
    """A [B, H, T, D] fp16 tensor on the cache's device as a tsa_rows: rows of consecutive elements,
    any other strides."""
    torch = _torch or _t()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is torch.float16 and t.get_device() == cache.index and t.shape == shape:
        b, h, r, d = t.stride()
        if d == 1:
            return _ROWS.pack(t.data_ptr(), b, h, r)
    raise ValueError(f"{name}: expected fp16 {tuple(shape)} on {cache.device} with consecutive row elements, got "
                     f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


def _counts(t, name, cache):
    torch = _torch or _t()
    if t.dtype is not torch.int32 or t.get_device() != cache.index or t.shape != cache.counts_shape or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {cache.B} on {cache.device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return t.data_ptr()


def _len(t, cache):
    if not isinstance(t, (_torch or _t()).Tensor):
        raise TypeError("len must be a torch.Tensor")
    return _counts(t, "len", cache)


def _kv8_call(fn, cache, stream, *args):
    """The entry point on the cache's device, made the current one for the call where it is another."""
    torch = _torch or _t()
    if torch._C._cuda_getDevice() == cache.index:
        _check(fn(cache._ref, *args, torch._C._cuda_getCurrentRawStream(cache.index) if stream is None else stream.cuda_stream))
    else:
        with torch.cuda.device(cache.index):
            _check(fn(cache._ref, *args, _stream(stream)))


def kv8_write(cache, k, v, len, n_new=None, stream=None):
    """Writes k, v [B, Hkv, T, D] fp16 (rows of consecutive elements, any other strides) at the end of
    each sequence: len [B] int32 counts its tokens, these among them; n_new [B] int32 (default T each)
    says how many of the T rows are tokens, the rest is padding."""
    T = k.shape[2]
    shape = (cache.B, cache.Hkv, T, cache.D)
    _kv8_call(load().tsa_kv8_write, cache, stream, _rows(k, shape, "k", cache), _rows(v, shape, "v", cache), _len(len, cache),
              None if n_new is None else _counts(n_new, "n_new", cache), T)


def kv8_read(cache, len, S=None, start=None, k_out=None, v_out=None, stream=None):
    """Positions start .. start + S - 1 of each sequence (start [B] int32, default 0) as fp16 k, v
    [B, Hkv, S, D]; rows of positions behind the sequence or without a page are left as they were
    (0 in outputs made here)."""
    torch = _torch or _t()
    if S is None:
        S = k_out.shape[2] if k_out is not None else v_out.shape[2] if v_out is not None else cache.max_len
    shape = (cache.B, cache.Hkv, S, cache.D)
    if k_out is None and v_out is None:
        k_out, v_out = (_zeros(shape, cache, stream) for _ in range(2))
    _kv8_call(load().tsa_kv8_read, cache, stream, _len(len, cache), None if start is None else _counts(start, "start", cache), S,
              None if k_out is None else _rows(k_out, shape, "k_out", cache),
              None if v_out is None else _rows(v_out, shape, "v_out", cache))
    return k_out, v_out


def _zeros(shape, cache, stream, dtype=None, value=0):
    """An output with a value where nothing will be written, filled on the stream that writes it."""
    torch = _torch or _t()
    s = torch.cuda.current_stream(cache.device) if stream is None else stream
    with torch.cuda.stream(s):
        return torch.full(shape, value, dtype=dtype or torch.float16, device=cache.device)


def _max_len(max_len, cache):
    """No sequence is longer than the cache, and a C int holds no more."""
    return cache.max_len if max_len is None or max_len > cache.max_len else max_len


def kv8_workspace_bytes(cache, T, Hq, max_len=None, top=0) -> int:
    """Workspace bytes of attn_kv8_fwd (top = 0), or of kv8_select and attn_kv8_blocks_fwd, which may
    share one (top > 0)."""
    return int(load().tsa_kv8_workspace_bytes(cache._ref, T, Hq, _max_len(max_len, cache), top))


def _queries(q, cache, gate, out, n_new, stream):
    """Views of q, gate and out, the output, and Hq, T; made before anything is launched."""
    if q.dim() != 4:
        raise ValueError(f"q: expected [B, Hq, T, D], got {tuple(q.shape)}")
    _, Hq, T, _ = q.shape
    shape = (cache.B, Hq, T, cache.D)
    qp = _rows(q, shape, "q", cache)
    gp = None if gate is None else _rows(gate, shape, "gate", cache)
    if out is None:
        if n_new is not None:
            out = _zeros(shape, cache, stream)
        elif stream is None:
            out = (_torch or _t()).empty(shape, dtype=q.dtype, device=cache.device)
        else:  # memory that no other stream's earlier work still uses
            with (_torch or _t()).cuda.stream(stream):
                out = _t().empty(shape, dtype=q.dtype, device=cache.device)
    return qp, gp, _rows(out, shape, "out", cache), out, Hq, T


def _ws(ws, cache, T, Hq, max_len, top, stream):
    """Pointer and bytes of the caller's workspace, or of one for this call (and the tensor itself, to
    be held until the call is made)."""
    if ws is None:
        ws = _scratch(kv8_workspace_bytes(cache, T, Hq, max_len, top), cache.device, stream)
    elif ws.get_device() != cache.index or not ws.is_contiguous():
        raise ValueError(f"ws: expected a contiguous tensor on {cache.device}, got one on {ws.device}")
    return ws.data_ptr(), ws.numel() * ws.element_size(), ws


def attn_kv8_fwd(q, cache, len, n_new=None, gate=None, out=None, scale=None, causal=True, max_len=None, ws=None,
                 stream=None):
    """Attention of q [B, Hq, T, D], the last n_new tokens of each sequence (default T each), over the
    cache that holds them already: softmax(scale q K^T) V over the keys up to each query's own
    (causal) or all len of them, times sigmoid(gate) if given.  Hq % Hkv == 0.  Rows of padding
    (t >= n_new) are left as they were (0 in an output made here).  max_len: no sequence is longer (a
    tighter split of the keys: results for longer ones are right too, their last bits may depend on it)."""
    qp, gp, op, out, Hq, T = _queries(q, cache, gate, out, n_new, stream)
    max_len = _max_len(max_len, cache)
    wp, wn, ws = _ws(ws, cache, T, Hq, max_len, 0, stream)
    _kv8_call(load().tsa_attn_kv8_fwd, cache, stream, qp, gp, op, _len(len, cache),
              None if n_new is None else _counts(n_new, "n_new", cache), T, Hq, max_len,
              1.0 / math.sqrt(cache.D) if scale is None else float(scale), 1 if causal else 0, wp, wn)
    return out


def _blocks(blocks, cache, T, top):
    torch = _torch or _t()
    if blocks.dtype is not torch.int32 or blocks.get_device() != cache.index or not blocks.is_contiguous() or \
            blocks.shape != (cache.B, cache.Hkv, T, top):
        raise ValueError(f"blocks: expected contiguous int32 {(cache.B, cache.Hkv, T, top)} on {cache.device}, got "
                         f"{tuple(blocks.shape)} {blocks.dtype} on {blocks.device}")
    return blocks.data_ptr()


def kv8_select(q, cache, len, top, n_new=None, first=1, recent=1, out=None, max_len=None, ws=None, stream=None):
    """The blocks [B, Hkv, T, top] int32 that each query of q [B, Hq, T, D] attends to: the first
    `first`, its own and the `recent` before it, and the best by score, ascending, -1 behind the last.
    Rows of padding are left as they were (-1 in an output made here).  max_len: no sequence is longer,
    nor becomes so in replays of a captured call (blocks behind it have no score and are chosen last)."""
    torch = _torch or _t()
    if q.dim() != 4:
        raise ValueError(f"q: expected [B, Hq, T, D], got {tuple(q.shape)}")
    _, Hq, T, _ = q.shape
    qp = _rows(q, (cache.B, Hq, T, cache.D), "q", cache)
    if min(top, first, recent) < -1 << 31 or max(top, first, recent) >= 1 << 31:
        raise ValueError(f"top = {top}, first = {first}, recent = {recent}: at least one is no 32-bit number")
    if out is None:
        out = _zeros((cache.B, cache.Hkv, T, top), cache, stream, torch.int32, -1)
    max_len = _max_len(max_len, cache)
    wp, wn, ws = _ws(ws, cache, T, Hq, max_len, top, stream)
    _kv8_call(load().tsa_kv8_select, cache, stream, qp, _len(len, cache),
              None if n_new is None else _counts(n_new, "n_new", cache), T, Hq, top, first, recent, _blocks(out, cache, T, top),
              max_len, wp, wn)
    return out


def attn_kv8_blocks_fwd(q, cache, len, blocks, n_new=None, gate=None, out=None, scale=None, ws=None, stream=None):
    """attn_kv8_fwd (causal) over the listed blocks [B, Hkv, T, top] only (of kv8_select, or the
    caller's own: entries that are no block up to the query's own are passed over, a block listed
    twice counts twice)."""
    qp, gp, op, out, Hq, T = _queries(q, cache, gate, out, n_new, stream)
    top = blocks.shape[-1]
    wp, wn, ws = _ws(ws, cache, T, Hq, 1, top, stream)
    _kv8_call(load().tsa_attn_kv8_blocks_fwd, cache, stream, qp, gp, op, _len(len, cache),
              None if n_new is None else _counts(n_new, "n_new", cache), T, Hq, _blocks(blocks, cache, T, top), top,
              1.0 / math.sqrt(cache.D) if scale is None else float(scale), wp, wn)
    return out


# ---------------------------------------------------------------------------------------
# rotary positions, and attention's training pair
# ---------------------------------------------------------------------------------------
ROPE_SCALINGS = (None, "linear", "ntk", "yarn", "wavelength")


class Rope:
    """Rotary positions of heads of D elements (include/tsa.h, tsa_rope): pairs of the first `rot`
    elements (default all) turn by position * base^(-2 i / rot), scaled by one of ROPE_SCALINGS.
    interleaved: pairs (2 i, 2 i + 1), otherwise (i, i + rot / 2).  Holds the table of frequencies on
    `device`."""

    def __init__(self, D, rot=None, base=10000.0, interleaved=False, scaling=None, factor=1.0, orig_len=0, beta_fast=32.0,
                 beta_slow=1.0, low=1.0, high=4.0, amp=None, device="cuda"):
        torch = _torch or _t()
        rot = D if rot is None else rot
        if D not in (64, 128, 256):
            raise ValueError(f"D must be 64, 128 or 256, got {D}")
        if rot < 2 or rot % 2 or rot > D:
            raise ValueError(f"rot must be even, 2 .. {D}, got {rot}")
        if scaling not in ROPE_SCALINGS:
            raise ValueError(f"scaling must be one of {ROPE_SCALINGS}, got {scaling!r}")
        if not 0 <= orig_len < 1 << 31:
            raise ValueError(f"orig_len is no 32-bit count: {orig_len}")
        params = TsaRopeParams(base, factor, beta_fast, beta_slow, low, high, rot, ROPE_SCALINGS.index(scaling), orig_len)
        table, found = (ctypes.c_uint64 * (rot // 2))(), ctypes.c_float()
        _check(load().tsa_rope_freqs(ctypes.addressof(params), ctypes.addressof(table), ctypes.addressof(found)))
        self.D, self.rot, self.interleaved = D, rot, bool(interleaved)
        self.amp = found.value if amp is None else float(amp)
        self.turns = [f * 2.0 ** -64 for f in table]
        # torch has few operations on uint64: the same bits as int64
        self.freq = torch.tensor([f - (1 << 64) if f >> 63 else f for f in table], dtype=torch.int64).to(device)
        if self.freq.device.type != "cuda":
            raise ValueError(f"a table of frequencies lies on a GPU, not on {device}")
        self.index = self.freq.get_device()
        self.view = TsaRopePlan(_ptr(self.freq), self.amp, rot, int(self.interleaved))
        self._ref = ctypes.byref(self.view)


_pack_rows = _ROWS.pack
_tensor = None  # torch.Tensor, once torch is there


def _rows_on(t, shape, name, index, dtype):
    """A [B, H, T, D] tensor on GPU `index` as a tsa_rows: rows of consecutive elements, any other strides."""
    if t.__class__ is not _tensor and not isinstance(t, (_torch or _t()).Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is dtype and t.shape == shape and t.get_device() == index:  # (index is a GPU's: not -1)
        b, h, r, d = t.stride()
        if d == 1:
            return _pack_rows(t.data_ptr(), b, h, r)
    raise ValueError(f"{name}: expected {dtype} {tuple(shape)} on GPU {index} with consecutive row elements, got "
                     f"{tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


def _ints_on(t, shape, name, index):
    """A contiguous int32 tensor on GPU `index`."""
    torch = _torch or _t()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not torch.int32 or not t.is_cuda or t.get_device() != index or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor of {tuple(shape)} on GPU {index}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")
    return t.data_ptr()


def _call_on(fn, index, stream, *args):
    """The entry point on GPU `index`, made the current one for the call where it is another."""
    torch = _torch or _t()
    if torch._C._cuda_getDevice() == index:
        _check(fn(*args, torch._C._cuda_getCurrentRawStream(index) if stream is None else stream.cuda_stream))
    else:
        with torch.cuda.device(index):
            _check(fn(*args, _stream(stream)))


def _new_like(x, padded, stream):
    """An output shaped and laid out like x, 0 where padding is left as it was, made on the stream that writes it."""
    torch = _torch or _t()
    make = torch.zeros_like if padded else torch.empty_like
    fmt = torch.preserve_format
    # an expanded input (stride 0) has no layout for an output
    if any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
        fmt = torch.contiguous_format
    if stream is None and torch._C._cuda_getDevice() == x.get_device():
        return make(x, memory_format=fmt)
    with torch.cuda.stream(torch.cuda.current_stream(x.device) if stream is None else stream):
        return make(x, memory_format=fmt)


def _four(t, name):
    global _tensor
    if t.__class__ is not _tensor:
        _tensor = (_torch or _t()).Tensor
        if not isinstance(t, _tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    shape = t.shape
    if shape.__len__() != 4 or not t.is_cuda:
        raise ValueError(f"{name}: expected a 4-d tensor on a GPU, got {tuple(shape)} on {t.device}")
    return shape


def _rope(rope, q, k, pos, len, n_new, q_out, k_out, back, stream):
    torch = _torch or _t()
    q_shape = B, Hq, T, D = _four(q, "q")
    i, dtype = rope.index, q.dtype
    if dtype is not torch.float16 and dtype is not torch.float32:
        raise ValueError(f"q: expected fp16 or fp32, got {dtype}")
    if D != rope.D:
        raise ValueError(f"q has heads of {D} elements, the rotation {rope.D}")
    q_in = _rows_on(q, q_shape, "q", i, dtype)
    if k is None:
        if k_out is not None:
            raise ValueError("k_out without k")
        Hk, k_in = 0, None
    else:
        Hk = _four(k, "k")[1]
        k_shape = (B, Hk, T, D)
        k_in = _rows_on(k, k_shape, "k", i, dtype)
        if k_out is None:
            k_out = _new_like(k, n_new is not None, stream)
    if q_out is None:
        q_out = _new_like(q, n_new is not None, stream)
    _call_on((_lib or load()).tsa_rope, i, stream, rope._ref, TSA_TYPE_F32 if dtype is torch.float32 else TSA_TYPE_F16, q_in,
             _rows_on(q_out, q_shape, "q_out", i, dtype), Hq, k_in, None if k is None else _rows_on(k_out, k_shape, "k_out", i, dtype),
             Hk, None if pos is None else _ints_on(pos, (B, T), "pos", i), None if len is None else _ints_on(len, (B,), "len", i),
             None if n_new is None else _ints_on(n_new, (B,), "n_new", i), B, T, D, back)
    return q_out, k_out


def rope_fwd(rope, q, k=None, pos=None, len=None, n_new=None, q_out=None, k_out=None, stream=None):
    """Rotates q [B, Hq, T, D] and k [B, Hk, T, D] (fp16 or fp32, rows of consecutive elements, any other
    strides) and returns (q_out, k_out); q_out may be q, k_out may be k.  Row t is at pos[b, t] (int32
    [B, T]), or at len[b] - n_new[b] + t (int32 [B]; the cache's len and n_new), or at t.  Rows behind
    n_new (default T) are left as they were (0 in outputs made here)."""
    return _rope(rope, q, k, pos, len, n_new, q_out, k_out, 0, stream)


def rope_bwd(rope, dq, dk=None, pos=None, len=None, n_new=None, q_out=None, k_out=None, stream=None):
    """The gradients of rope_fwd's q and k from those of its outputs, with the same positions."""
    return _rope(rope, dq, dk, pos, len, n_new, q_out, k_out, 1, stream)


def _train_shapes(q, k, v, gate, len_q, len_k):
    torch = _torch or _t()
    B, Hq, Tq, D = _four(q, "q")
    _, Hkv, Tk, _ = _four(k, "k")
    i, half = q.get_device(), torch.float16
    views = (_rows_on(q, q.shape, "q", i, half), _rows_on(k, (B, Hkv, Tk, D), "k", i, half), _rows_on(v, (B, Hkv, Tk, D), "v", i, half),
             None if gate is None else _rows_on(gate, q.shape, "gate", i, half))
    lens = (None if len_q is None else _ints_on(len_q, (B,), "len_q", i), None if len_k is None else _ints_on(len_k, (B,), "len_k", i))
    return views, lens, (B, Hq, Hkv, Tq, Tk, D)


def _stat(lse, shape, name, index):
    torch = _torch or _t()
    if not isinstance(lse, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if lse.dtype is not torch.float32 or not lse.is_cuda or lse.get_device() != index or lse.shape != shape or not lse.is_contiguous():
        raise ValueError(f"{name}: expected contiguous fp32 {tuple(shape)} on GPU {index}, got {tuple(lse.shape)} {lse.dtype} on {lse.device}")
    return lse.data_ptr()


def attn_train_fwd(q, k, v, gate=None, len_q=None, len_k=None, out=None, lse=None, scale=None, causal=True, stream=None):
    """The forward pass that attn_bwd goes back from: returns (o, lse) for q, gate [B, Hq, Tq, D] and k, v
    [B, Hkv, Tk, D] fp16 (rows of consecutive elements, any other strides), o = softmax(scale q K^T) V, times
    sigmoid(gate) if given, lse [B, Hq, Tq] fp32 the logarithms of the softmax sums.  len_q, len_k (int32
    [B], default Tq, Tk) count each sequence's rows; under the causal mask query t sees keys up to
    t + len_k - len_q.  Rows of padding are left as they were (0 in outputs made here)."""
    torch = _torch or _t()
    views, lens, (B, Hq, Hkv, Tq, Tk, D) = _train_shapes(q, k, v, gate, len_q, len_k)
    i = q.get_device()
    if out is None:
        out = _new_like(q, len_q is not None, stream)
    op = _rows_on(out, q.shape, "out", i, torch.float16)
    if lse is None:
        with torch.cuda.stream(torch.cuda.current_stream(q.device) if stream is None else stream):
            lse = torch.zeros(B, Hq, Tq, dtype=torch.float32, device=q.device)
    _call_on((_lib or load()).tsa_attn_train_fwd, i, stream, *views, op, _stat(lse, (B, Hq, Tq), "lse", i), *lens, B, Hq, Hkv, Tq, Tk, D,
             1.0 / math.sqrt(D) if scale is None else float(scale), 1 if causal else 0)
    return out, lse


def attn_bwd_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, gated=False, causal=True) -> int:
    """Workspace bytes of one attn_bwd call."""
    return int(load().tsa_attn_bwd_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, 1 if gated else 0, 1 if causal else 0))


def attn_bwd(d_out, q, k, v, out, lse, gate=None, len_q=None, len_k=None, dq=None, dk=None, dv=None, dgate=None, scale=None,
             causal=True, ws=None, stream=None):
    """The gradients (dq, dk, dv, dgate; dgate None without a gate) for the gradient d_out of attn_train_fwd's
    o, from its o and lse and the arguments it had.  Shared key and value heads get the sum over their
    query heads.  Rows of padding are left as they were (0 in outputs made here).  Outputs lie on no input."""
    torch = _torch or _t()
    views, lens, (B, Hq, Hkv, Tq, Tk, D) = _train_shapes(q, k, v, gate, len_q, len_k)
    i, half = q.get_device(), torch.float16
    if gate is None and dgate is not None:
        raise ValueError("dgate without gate")
    gp, op = _rows_on(d_out, q.shape, "d_out", i, half), _rows_on(out, q.shape, "out", i, half)
    lp = _stat(lse, (B, Hq, Tq), "lse", i)
    dq = _new_like(q, len_q is not None, stream) if dq is None else dq
    dk = _new_like(k, len_k is not None, stream) if dk is None else dk
    dv = _new_like(v, len_k is not None, stream) if dv is None else dv
    if gate is not None and dgate is None:
        dgate = _new_like(gate, len_q is not None, stream)
    grads = (_rows_on(dq, q.shape, "dq", i, half), _rows_on(dk, k.shape, "dk", i, half), _rows_on(dv, v.shape, "dv", i, half),
             None if gate is None else _rows_on(dgate, q.shape, "dgate", i, half))
    if ws is None:
        ws = _scratch(attn_bwd_workspace_bytes(B, Hq, Hkv, Tq, Tk, D, gate is not None, causal), q.device, stream)
    elif not ws.is_cuda or ws.get_device() != i or not ws.is_contiguous():
        raise ValueError(f"ws: expected a contiguous tensor on GPU {i}, got one on {ws.device}")
    _call_on((_lib or load()).tsa_attn_bwd, i, stream, gp, *views, op, lp, *grads, *lens, B, Hq, Hkv, Tq, Tk, D,
             1.0 / math.sqrt(D) if scale is None else float(scale), 1 if causal else 0, _ptr(ws), ws.numel() * ws.element_size())
    return dq, dk, dv, dgate
