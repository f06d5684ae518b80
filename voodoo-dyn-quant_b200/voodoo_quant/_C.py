"""ctypes binding of libvoodoo_b200.so (the sm_100a kernels) for torch tensors.

The library is loaded from this package directory (built in-tree by
``__graft_entry__.build()``).  There is no fallback: if the library is
missing, or CUDA is not available, every entry point raises ``RuntimeError``.
Status codes of the C ABI map onto the reference's exception conventions:
invalid shapes / alignment / unknown quant types raise ``ValueError``
(voodoo_quant/ggml.py:161-164,195-198,242-253 in the reference), CUDA
failures raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import functools
import math
import os
from array import array
from operator import attrgetter
from pathlib import Path

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

LIB_NAME = "libvoodoo_b200.so"
LIB_PATH = Path(__file__).resolve().parent / LIB_NAME

VQ_ERR_INVALID = -1
VQ_ERR_CUDA = -2
VQ_ERR_UNSUPPORTED = -3

# ggml type ids of the supported candidate formats.
GGML_TYPE = {"Q8_0": 8, "Q2_K": 10, "Q3_K": 11, "Q4_K": 12, "Q5_K": 13, "Q6_K": 14, "IQ4_XS": 23}

_lib = None

_i64 = ctypes.c_int64
_vp = ctypes.c_void_p
_int = ctypes.c_int
_f32 = ctypes.c_float


def _declare(lib):
    sig = {
        "vq_last_error": (ctypes.c_char_p, []),
        "vq_abi_version": (_int, []),
        "vq_format_info": (_int, [_int, ctypes.POINTER(_int), ctypes.POINTER(_int)]),
        "vq_device_error": (_int, [_vp, ctypes.POINTER(_int)]),
        "vq_device_error_async": (_int, [_vp, _vp]),
        "vq_dequant": (_int, [_int, _vp, _i64, _i64, _vp, _vp]),
        "vq_quantize": (_int, [_int, _vp, _int, _i64, _i64, _i64, _vp, _vp]),
        "vq_mix": (_int, [_int, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp]),
        "vq_linear_fwd": (_int, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _vp]),
        "vq_linear_fwd_swiglu": (_int, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _vp]),
        "vq_set_gategrad_sm_reserve": (_int, [_int]),
        "vq_set_gemm_sm_reserve": (_int, [_int]),
        "vq_route_prep": (_int, [_vp, _i64, _int, _vp, _vp, _vp, _vp]),
        "vq_linear_fwd_grouped": (_int, [_vp, _i64, _i64, _i64, _int, _vp, _i64, _i64, _vp, _vp, _i64, _vp]),
        "vq_linear_dx": (_int, [_vp, _i64, _i64, _i64, _vp, _i64, _i64, _vp, _i64, _vp]),
        "vq_gategrad_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _int]),
        "vq_gategrad": (_int, [_vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp, _vp, _i64, _vp,
                               ctypes.c_size_t, _vp, _vp]),
        "vq_gategrad_noalloc": (_int, [_vp, _i64, _vp, _i64, _i64, _i64, _i64, _int, _vp, _vp, _i64, _vp, _vp]),
        "vq_gategrad_grouped_workspace_bytes": (ctypes.c_size_t, [_i64, _i64, _int, _int]),
        "vq_gategrad_grouped": (_int, [_vp, _i64, _vp, _i64, _i64, _int, _vp, _i64, _int, _vp, _vp, _i64, _vp,
                                       ctypes.c_size_t, _vp, _i64, _vp]),
        "vq_mixgemm_fwd": (_int, [_vp, _i64, _i64, _i64, _int, _vp, _vp, _vp, _i64, _i64, _vp, _i64, _vp,
                                  _i64, _vp]),
        "vq_mixgemm_fwd_fused": (_int, [_vp, _i64, _i64, _i64, _int, _vp, _vp, _vp, _i64, _i64, _vp, _i64,
                                        _vp]),
        "vq_mixgemm_dx": (_int, [_vp, _i64, _i64, _i64, _int, _vp, _vp, _vp, _i64, _i64, _vp, _i64, _vp,
                                 _i64, _vp]),
        "vq_loss_fused": (_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _f32, _f32, _f32, _vp, _vp, _vp,
                                 _i64, _vp]),
        "vq_loss_stats": (_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _f32, _vp, _vp]),
        "vq_loss_combine": (_int, [_vp, _int, _i64, _f32, _vp, _vp, _vp, _vp]),
        "vq_loss_grad": (_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _f32, _vp, _f32, _f32, _vp,
                                _i64, _vp]),
        "vq_rmsnorm_fwd": (_int, [_vp, _i64, _i64, _i64, _vp, _f32, _vp, _i64, _vp, _vp]),
        "vq_rmsnorm_bwd": (_int, [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _i64, _vp]),
        "vq_add_rmsnorm_fwd": (_int, [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _f32, _vp, _i64, _vp, _i64, _vp, _vp]),
        "vq_rmsnorm_bwd_add": (_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _i64, _vp]),
        "vq_rope": (_int, [_vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _int, _vp, _vp, _vp]),
        "vq_swiglu_fwd": (_int, [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp]),
        "vq_swiglu_bwd": (_int, [_vp, _i64, _vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _i64, _vp]),
        "vq_qk_norm_rope_fwd": (_int, [_vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp, _int, _vp, _vp, _vp, _int, _i64, _i64,
                                       _i64, _i64, _f32, _f32, _int, _vp, _vp, _vp]),
        "vq_qk_norm_rope_workspace_bytes": (ctypes.c_size_t, [_i64]),
        "vq_qk_norm_rope_bwd": (_int, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp, _int, _vp, _vp, _vp,
                                       _int, _i64, _i64, _i64, _i64, _f32, _f32, _int, _vp, _vp, _vp, _vp, _vp,
                                       ctypes.c_size_t, _vp]),
        "vq_embed_plan_bytes": (ctypes.c_size_t, [_i64]),
        "vq_embed_plan": (_int, [_vp, _int, _i64, _i64, _i64, _vp, ctypes.c_size_t, _vp]),
        "vq_embed_mix": (_int, [_int, _vp, _vp, _vp, _vp, _int, _i64, _vp, ctypes.c_size_t, _i64, _i64, _i64, _i64, _f32,
                                _int, _vp, _i64, _vp]),
        "vq_embed_gategrad_workspace_bytes": (ctypes.c_size_t, [_int]),
        "vq_embed_gategrad": (_int, [_int, _vp, _vp, _vp, ctypes.c_size_t, _i64, _i64, _i64, _i64, _f32, _vp, _i64, _int,
                                     _vp, ctypes.c_size_t, _vp, _vp]),
        "vq_clip_grad_norm_workspace_bytes": (ctypes.c_size_t, [_int]),
        "vq_clip_grad_norm": (_int, [_int, _vp, _vp, _vp, _f32, _int, _vp, ctypes.c_size_t, _vp, _vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return sig.keys()


EXPORTED = (
    "vq_last_error", "vq_abi_version", "vq_format_info", "vq_device_error", "vq_device_error_async", "vq_dequant", "vq_mix",
    "vq_linear_fwd", "vq_linear_fwd_swiglu", "vq_linear_fwd_grouped", "vq_set_gategrad_sm_reserve", "vq_set_gemm_sm_reserve", "vq_quantize", "vq_route_prep", "vq_linear_dx", "vq_gategrad_workspace_bytes", "vq_gategrad", "vq_gategrad_noalloc",
    "vq_gategrad_grouped_workspace_bytes", "vq_gategrad_grouped",
    "vq_mixgemm_fwd", "vq_mixgemm_fwd_fused", "vq_mixgemm_dx",
    "vq_loss_fused", "vq_loss_stats", "vq_loss_combine", "vq_loss_grad",
    "vq_rmsnorm_fwd", "vq_rmsnorm_bwd", "vq_add_rmsnorm_fwd", "vq_rmsnorm_bwd_add", "vq_rope", "vq_swiglu_fwd", "vq_swiglu_bwd",
    "vq_qk_norm_rope_fwd", "vq_qk_norm_rope_workspace_bytes", "vq_qk_norm_rope_bwd",
    "vq_embed_plan_bytes", "vq_embed_plan", "vq_embed_mix", "vq_embed_gategrad_workspace_bytes", "vq_embed_gategrad",
    "vq_clip_grad_norm_workspace_bytes", "vq_clip_grad_norm",
)


def load_library(path: str | os.PathLike | None = None):
    """Load (once) and return the ctypes handle; raises RuntimeError if absent."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path is not None else LIB_PATH
    if not p.exists():
        raise RuntimeError(
            f"{LIB_NAME} not found at {p}; build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "(the B200 path has no CPU fallback)"
        )
    lib = ctypes.CDLL(str(p))
    _declare(lib)
    if path is None:
        _lib = lib
    return lib


def _check(rc: int) -> None:
    if rc == 0:
        return
    msg = _lib.vq_last_error().decode(errors="replace")
    if rc in (VQ_ERR_INVALID, VQ_ERR_UNSUPPORTED):
        raise ValueError(msg)
    raise RuntimeError(f"libvoodoo_b200: {msg}")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _raw_stream(device_index: int) -> int:
    """Current stream's handle on a device, without the Python stream object (a few microseconds of a short call)."""
    return torch._C._cuda_getCurrentRawStream(device_index)


def _require_cuda(*ts: torch.Tensor) -> None:
    load_library()
    for t in ts:
        if not t.is_cuda:
            raise RuntimeError("libvoodoo_b200 kernels need CUDA tensors (no CPU fallback)")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def no_tangents(what: str, ts) -> None:
    """Refuses forward-mode duals, whose tangents a kernel that gets the values' pointers would lose without a word.
    (An autograd function without a ``jvp`` refuses them itself, but only where one is applied.)"""
    if forward_ad._current_level >= 0:  # some level is open: rarely
        for t in ts:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: no forward-mode derivative (a tensor carries a tangent)")


def first_order(backward):
    """``once_differentiable`` for a Function's backward, without its bookkeeping where no graph of the gradients is
    built (7 us of the 140 of a short forward and backward: the engine's thread finds the interpreter's data cold)."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        no_tangents("backward", grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


# dtype codes of the entry points that take more than one floating type
_FLOAT_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _float_code(t: torch.Tensor, name: str) -> int:
    code = _FLOAT_CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: float32, bfloat16 or float16 expected, got {t.dtype}")
    return code


def _device_of(*ts: torch.Tensor) -> int:
    """Index of the CUDA device that all of the tensors are on."""
    d = ts[0].get_device()
    for t in ts:
        if t.get_device() != d or d < 0:
            _require_cuda(*ts)
            raise ValueError(f"tensors on one device expected, got {[str(u.device) for u in ts]}")
    if _lib is None:
        load_library()
    return d


def format_info(qtype: str) -> tuple[int, int]:
    lib = load_library()
    be, bb = _int(), _int()
    rc = lib.vq_format_info(GGML_TYPE.get(qtype, -1), ctypes.byref(be), ctypes.byref(bb))
    _check(rc)
    return be.value, bb.value


@functools.cache
def _workspace_bytes(entry: str, n: int) -> int:
    """What a workspace entry point says for a size."""
    return getattr(_lib, entry)(n)


_GEOMETRY: dict[str, tuple[int, int]] = {}


def _geometry(qtype: str) -> tuple[int, int]:
    """``format_info`` of a supported type, looked up once."""
    g = _GEOMETRY.get(qtype)
    if g is None:
        if qtype not in GGML_TYPE:
            raise ValueError(f"Unknown quant type: {qtype}. Supported: {list(GGML_TYPE)}")
        g = _GEOMETRY[qtype] = format_info(qtype)
    return g


def device_error(device: torch.device | None = None) -> int:
    """Synchronise the current stream and return/clear the device error word."""
    lib = load_library()
    code = _int()
    st = torch.cuda.current_stream(device).cuda_stream
    _check(lib.vq_device_error(st, ctypes.byref(code)))
    return code.value


_ERROR_TEXT = {1: "a kernel gave up waiting", 2: "unknown block format", 3: "misaligned shared memory",
               4: "token id outside the embedding table", 5: "a lookup met the plan of other token ids"}


def device_error_text(code: int) -> str:
    return f"{_ERROR_TEXT.get(code >> 16, 'unknown error')} (device error word {code:#x})"


class ErrorWatch:
    """Reads the devices' error words behind each step's work without making the host wait for that step: ``poll``
    raises what the kernels up to the poll before it reported, ``check`` what all of them did.  The word is cleared."""

    def __init__(self, devices):
        self._devices = [torch.device(d) for d in devices]
        self._pending = []  # (word on the host, event behind its copy) of the poll before

    def poll(self) -> None:
        before, self._pending = self._pending, []
        for d in self._devices:
            with torch.cuda.device(d):
                word = torch.empty(1, dtype=torch.int32, device=d)
                _check(load_library().vq_device_error_async(word.data_ptr(), _raw_stream(d.index)))
                word, event = word.to("cpu", non_blocking=True), torch.cuda.Event()
                event.record()
                self._pending.append((word, event))
        for word, event in before:
            event.synchronize()
            if int(word):
                self.check()

    def check(self) -> None:
        self._pending = []
        codes = {}
        for d in self._devices:
            with torch.cuda.device(d):
                codes[d] = device_error()
        for d, code in codes.items():
            if code:
                raise RuntimeError(f"{d}: {device_error_text(code)}")


def quantize(w: torch.Tensor, qtype: str) -> torch.Tensor:
    """GPU quantiser: float32 / bfloat16 [rows, cols] -> uint8 [rows * cols / 32, 34] Q8_0 blocks
    (byte-identical to ggml's reference rule); other types raise ValueError."""
    _require_cuda(w)
    if qtype not in GGML_TYPE:
        raise ValueError(f"Unknown quant type: {qtype}. Supported: {list(GGML_TYPE)}")
    if w.dim() != 2:
        raise ValueError(f"quantize expects a 2-D weight, got shape {tuple(w.shape)}")
    if w.dtype not in (torch.float32, torch.bfloat16):
        w = w.to(torch.float32)
    if w.stride(1) != 1:
        w = w.contiguous()
    be, bb = format_info(qtype)
    rows, cols = w.shape
    out = torch.empty(rows * (cols // be) if cols % be == 0 else 0, bb, dtype=torch.uint8, device=w.device)
    _check(_lib.vq_quantize(GGML_TYPE[qtype], w.data_ptr(), 0 if w.dtype == torch.float32 else 1, rows, cols,
                            w.stride(0), out.data_ptr(), _stream(w)))
    return out


def dequant(qbytes: torch.Tensor, qtype: str, rows: int, cols: int) -> torch.Tensor:
    """Bit-exact decode of packed blocks -> float32 [rows, cols] on the blocks' device."""
    _require_cuda(qbytes)
    if qtype not in GGML_TYPE:
        raise ValueError(f"Unknown quant type: {qtype}. Supported: {list(GGML_TYPE)}")
    be, bb = format_info(qtype)
    if cols % be:
        raise ValueError(f"{qtype} requires in_features % {be} == 0, got {cols}")
    if qbytes.numel() != rows * (cols // be) * bb:
        raise ValueError(
            f"qweight size {qbytes.numel()} does not match {rows * (cols // be)} blocks of {bb} bytes for {qtype}"
        )
    qb = qbytes.contiguous()
    out = torch.empty(rows, cols, dtype=torch.float32, device=qb.device)
    _check(_lib.vq_dequant(GGML_TYPE[qtype], qb.data_ptr(), rows, cols, out.data_ptr(), _stream(qb)))
    return out


def _cand_arrays(qtypes, qbytes):
    K = len(qtypes)
    types = (_int * K)(*[GGML_TYPE[q] for q in qtypes])
    ptrs = (_vp * K)(*[q.data_ptr() for q in qbytes])
    return K, types, ptrs


def mix(qtypes, qbytes, probs: torch.Tensor, rows: int, padded_cols: int, cols: int,
        out: torch.Tensor | None = None) -> torch.Tensor:
    """W_mix = sum_k probs[k] W_k -> bf16 [rows, ld] with ld = cols rounded up to 8."""
    _require_cuda(probs, *qbytes)
    ld = (cols + 7) // 8 * 8
    if out is None:
        out = torch.empty(rows, ld, dtype=torch.bfloat16, device=probs.device)
    K, types, ptrs = _cand_arrays(qtypes, qbytes)
    p = probs.detach().to(torch.float32).contiguous()
    _check(_lib.vq_mix(K, types, ptrs, p.data_ptr(), rows, padded_cols, cols, out.data_ptr(), out.stride(0),
                       _stream(p)))
    return out


def _as_operand(x: torch.Tensor) -> torch.Tensor:
    """bf16, unit column stride, leading dimension a multiple of 8, 16B-aligned base."""
    x = x.to(torch.bfloat16)
    if x.stride(-1) != 1 or x.stride(0) % 8 != 0 or x.data_ptr() % 16 != 0:
        cols = x.shape[1]
        ld = (cols + 7) // 8 * 8
        buf = torch.zeros(x.shape[0], ld, dtype=torch.bfloat16, device=x.device)
        buf[:, :cols] = x
        return buf
    return x


def linear_fwd(x: torch.Tensor, w: torch.Tensor, n_out: int | None = None, in_features: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """y[T, N] = x[T, Kin] w[N, Kin]^T in bf16 with fp32 accumulation."""
    _require_cuda(x, w)
    kin = x.shape[1] if in_features is None else in_features
    N = w.shape[0] if n_out is None else n_out
    x = _as_operand(x)
    if out is None:
        out = torch.empty(x.shape[0], N, dtype=torch.bfloat16, device=x.device)
    _check(_lib.vq_linear_fwd(x.data_ptr(), x.shape[0], kin, x.stride(0), w.data_ptr(), N, w.stride(0),
                              out.data_ptr(), out.stride(0), _stream(x)))
    return out


def mixgemm_fwd_fused(x: torch.Tensor, qtypes, qbytes, probs: torch.Tensor, n_out: int, padded_cols: int,
                      in_features: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W_mix^T with the mixture decoded into the GEMM's operand tiles
    (vq_mixgemm_fwd_fused); equal to ``mix`` then ``linear_fwd``."""
    _require_cuda(x, probs, *qbytes)
    kin = x.shape[1] if in_features is None else in_features
    x = _as_operand(x)
    K, types, ptrs = _cand_arrays(qtypes, qbytes)
    p = probs.to(torch.float32).contiguous()
    if out is None:
        out = torch.empty(x.shape[0], n_out, dtype=torch.bfloat16, device=x.device)
    _check(_lib.vq_mixgemm_fwd_fused(x.data_ptr(), x.shape[0], kin, x.stride(0), K, types, ptrs, p.data_ptr(), n_out,
                                     padded_cols, out.data_ptr(), out.stride(0), _stream(x)))
    return out


def linear_fwd_swiglu(x: torch.Tensor, w: torch.Tensor, F: int, in_features: int | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """h[T, F] = silu(x w[:F]^T) * (x w[F:2F]^T) in one GEMM (gate|up rounded
    to bf16 before the activation); T > 128 and F a multiple of 128."""
    _require_cuda(x, w)
    kin = x.shape[1] if in_features is None else in_features
    x = _as_operand(x)
    if out is None:
        out = torch.empty(x.shape[0], F, dtype=torch.bfloat16, device=x.device)
    _check(_lib.vq_linear_fwd_swiglu(x.data_ptr(), x.shape[0], kin, x.stride(0), w.data_ptr(), F, w.stride(0),
                                     out.data_ptr(), out.stride(0), _stream(x)))
    return out


def linear_fwd_grouped(x: torch.Tensor, ws: list, n_out: int, in_features: int, group_off: torch.Tensor,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """y[rows of group g] = x[rows of group g] ws[g]^T; group_off (int32, device, G + 1) need not be on the host."""
    _require_cuda(x, *ws)
    x = _as_operand(x)
    G = len(ws)
    ptrs = (_vp * G)(*[w.data_ptr() for w in ws])
    if out is None:
        out = torch.empty(x.shape[0], n_out, dtype=torch.bfloat16, device=x.device)
    go = group_off.to(torch.int32).contiguous()
    _check(_lib.vq_linear_fwd_grouped(x.data_ptr(), x.shape[0], in_features, x.stride(0), G, ptrs, n_out,
                                      ws[0].stride(0), go.data_ptr(), out.data_ptr(), out.stride(0), _stream(x)))
    return out


def linear_dx(dy: torch.Tensor, w: torch.Tensor, in_features: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """dx[T, Kin] = dy[T, N] w[N, Kin]."""
    _require_cuda(dy, w)
    dy = _as_operand(dy)
    N = w.shape[0]
    if out is None:
        out = torch.empty(dy.shape[0], in_features, dtype=torch.bfloat16, device=dy.device)
    _check(_lib.vq_linear_dx(dy.data_ptr(), dy.shape[0], N, dy.stride(0), w.data_ptr(), in_features, w.stride(0),
                             out.data_ptr(), out.stride(0), _stream(dy)))
    return out


def route_prep(keys: torch.Tensor, K: int):
    """(order int64 [T], inv int64 [T], group_off int32 [K + 1]) of the stable grouping of uint8 keys."""
    _require_cuda(keys)
    keys = keys.to(torch.uint8).contiguous().reshape(-1)
    T = keys.numel()
    order = torch.empty(T, dtype=torch.int64, device=keys.device)
    inv = torch.empty(T, dtype=torch.int64, device=keys.device)
    off = torch.empty(K + 1, dtype=torch.int32, device=keys.device)
    _check(_lib.vq_route_prep(keys.data_ptr(), T, K, order.data_ptr(), inv.data_ptr(), off.data_ptr(), _stream(keys)))
    return order, inv, off


def set_gategrad_sm_reserve(sms: int) -> None:
    """SMs later gate-gradient GEMMs leave free for a concurrent collective (0 = none)."""
    _check(load_library().vq_set_gategrad_sm_reserve(int(sms)))


def set_gemm_sm_reserve(sms: int) -> None:
    """SMs later forward / dX GEMMs leave free for a concurrent collective (0 = none)."""
    _check(load_library().vq_set_gemm_sm_reserve(int(sms)))


def gategrad(dy: torch.Tensor, x: torch.Tensor, qtypes, qbytes, n_out: int, in_features: int, padded_cols: int,
             workspace: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """grad_probs[k] = <dy^T x, W_k> (float32 [K], into `out` when given); dW is never materialised."""
    _require_cuda(dy, x, *qbytes)
    dy = _as_operand(dy)
    x = _as_operand(x)
    K, types, ptrs = _cand_arrays(qtypes, qbytes)
    need = _lib.vq_gategrad_workspace_bytes(n_out, in_features, K)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 4), dtype=torch.uint8, device=x.device)
    if out is None:
        g = torch.empty(K, dtype=torch.float32, device=x.device)
    else:
        if out.dtype != torch.float32 or out.numel() != K or not out.is_contiguous():
            raise ValueError("gategrad: out must be a contiguous float32 tensor of K elements")
        g = out
    _check(_lib.vq_gategrad(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), x.shape[0], n_out, in_features,
                            K, types, ptrs, padded_cols, workspace.data_ptr(), workspace.numel(), g.data_ptr(),
                            _stream(x)))
    return g


def gategrad_noalloc(dy: torch.Tensor, x: torch.Tensor, qtypes, qbytes, n_out: int, in_features: int,
                     padded_cols: int) -> torch.Tensor:
    """``gategrad`` on the library's own fixed scratch (vq_gategrad_noalloc), for
    callers that cannot allocate device scratch; the result still needs a [K]
    output tensor.  Calls that overlap on the GPU race on the shared scratch."""
    _require_cuda(dy, x, *qbytes)
    dy = _as_operand(dy)
    x = _as_operand(x)
    K, types, ptrs = _cand_arrays(qtypes, qbytes)
    g = torch.empty(K, dtype=torch.float32, device=x.device)
    _check(_lib.vq_gategrad_noalloc(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), x.shape[0], n_out,
                                    in_features, K, types, ptrs, padded_cols, g.data_ptr(), _stream(x)))
    return g


def gategrad_workspace_bytes(n_out: int, in_features: int, K: int) -> int:
    return int(load_library().vq_gategrad_workspace_bytes(n_out, in_features, K))


def gategrad_grouped_workspace_bytes(n_total: int, in_features: int, G: int, K: int) -> int:
    return int(load_library().vq_gategrad_grouped_workspace_bytes(n_total, in_features, G, K))


def gategrad_grouped(dy: torch.Tensor, x: torch.Tensor, qtypes, qbytes_per_layer, rows, in_features: int,
                     padded_cols: int, workspace: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """grad[g, k] = <dy_g^T x, W_{g,k}> for layers g side by side in dy's
    columns (rows[g] each, a multiple of 32), all with the formats `qtypes`:
    one gate-gradient GEMM (float32 [G, K], into `out` -- rows K floats
    apart or further, unit column stride -- when given)."""
    G = len(rows)
    _require_cuda(dy, x, *[b for bs in qbytes_per_layer for b in bs])
    dy = _as_operand(dy)
    x = _as_operand(x)
    K = len(qtypes)
    types = (_int * K)(*[GGML_TYPE[q] for q in qtypes])
    ptrs = (_vp * (G * K))(*[b.data_ptr() for bs in qbytes_per_layer for b in bs])
    rws = (ctypes.c_int64 * G)(*[int(r) for r in rows])
    need = _lib.vq_gategrad_grouped_workspace_bytes(sum(rows), in_features, G, K)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 4), dtype=torch.uint8, device=x.device)
    if out is None:
        out = torch.empty(G, K, dtype=torch.float32, device=x.device)
    elif out.dtype != torch.float32 or out.dim() != 2 or tuple(out.shape) != (G, K) or out.stride(1) != 1:
        raise ValueError("gategrad_grouped: out must be float32 [G, K] with unit column stride")
    _check(_lib.vq_gategrad_grouped(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), x.shape[0], G, rws,
                                    in_features, K, types, ptrs, padded_cols, workspace.data_ptr(), workspace.numel(),
                                    out.data_ptr(), out.stride(0), _stream(x)))
    return out


def loss_fused(s: torch.Tensor, t: torch.Tensor, targets: torch.Tensor, temperature: float, ce_weight: float,
               kl_weight: float, want_grad: bool = True):
    """Row CE, row T^2*KL and (optionally) d/ds for bf16 logits [rows, V]."""
    _require_cuda(s, t, targets)
    s = s.to(torch.bfloat16)
    t = t.to(torch.bfloat16)
    if s.stride(-1) != 1:
        s = s.contiguous()
    if t.stride(-1) != 1:
        t = t.contiguous()
    y = targets.to(torch.int64).contiguous()
    rows, V = s.shape
    ce = torch.empty(rows, dtype=torch.float32, device=s.device)
    kl = torch.empty(rows, dtype=torch.float32, device=s.device)
    g = torch.empty(rows, V, dtype=torch.bfloat16, device=s.device) if want_grad else None
    _check(_lib.vq_loss_fused(s.data_ptr(), s.stride(0), t.data_ptr(), t.stride(0), y.data_ptr(), rows, V,
                              float(temperature), float(ce_weight), float(kl_weight), ce.data_ptr(), kl.data_ptr(),
                              _ptr(g), g.stride(0) if g is not None else V, _stream(s)))
    return ce, kl, g


def loss_stats(s: torch.Tensor, t: torch.Tensor, targets: torch.Tensor, vocab_start: int, temperature: float):
    _require_cuda(s, t, targets)
    s = s.to(torch.bfloat16)
    t = t.to(torch.bfloat16)
    y = targets.to(torch.int64).contiguous()
    rows, V = s.shape
    st = torch.empty(rows, 8, dtype=torch.float32, device=s.device)
    _check(_lib.vq_loss_stats(s.data_ptr(), s.stride(0), t.data_ptr(), t.stride(0), y.data_ptr(), vocab_start, rows,
                              V, float(temperature), st.data_ptr(), _stream(s)))
    return st


def loss_combine(stats: torch.Tensor, temperature: float):
    """stats [R, rows, 8] -> (row_lse [rows, 4], row_ce [rows], row_kl [rows])."""
    _require_cuda(stats)
    stats = stats.to(torch.float32).contiguous()
    R, rows = stats.shape[0], stats.shape[1]
    lse = torch.empty(rows, 4, dtype=torch.float32, device=stats.device)
    ce = torch.empty(rows, dtype=torch.float32, device=stats.device)
    kl = torch.empty(rows, dtype=torch.float32, device=stats.device)
    _check(_lib.vq_loss_combine(stats.data_ptr(), R, rows, float(temperature), lse.data_ptr(), ce.data_ptr(),
                                kl.data_ptr(), _stream(stats)))
    return lse, ce, kl


def loss_grad(s: torch.Tensor, t: torch.Tensor, targets: torch.Tensor, vocab_start: int, temperature: float,
              row_lse: torch.Tensor, ce_weight: float, kl_weight: float) -> torch.Tensor:
    _require_cuda(s, t, targets, row_lse)
    s = s.to(torch.bfloat16)
    t = t.to(torch.bfloat16)
    y = targets.to(torch.int64).contiguous()
    rows, V = s.shape
    g = torch.empty(rows, V, dtype=torch.bfloat16, device=s.device)
    _check(_lib.vq_loss_grad(s.data_ptr(), s.stride(0), t.data_ptr(), t.stride(0), y.data_ptr(), vocab_start, rows,
                             V, float(temperature), row_lse.contiguous().data_ptr(), float(ce_weight),
                             float(kl_weight), g.data_ptr(), g.stride(0), _stream(s)))
    return g


# ---------------------------------------------------------------- Llama block elementwise
def _rows_operand(t: torch.Tensor) -> torch.Tensor:
    """bf16 2-D view with unit column stride, 16-byte aligned rows."""
    t = t.to(torch.bfloat16)
    if t.stride(-1) != 1 or t.stride(0) % 8 != 0 or t.data_ptr() % 16 != 0:
        t = t.contiguous()
    return t


def rmsnorm_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float):
    """(y [rows, D] bf16, rstd [rows] float32) for x [rows, D]."""
    _require_cuda(x, weight)
    x = _rows_operand(x)
    w = weight.to(torch.bfloat16).contiguous()
    rows, D = x.shape
    y = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    _check(_lib.vq_rmsnorm_fwd(x.data_ptr(), x.stride(0), rows, D, w.data_ptr(), float(eps), y.data_ptr(), y.stride(0),
                               rstd.data_ptr(), _stream(x)))
    return y, rstd


def rmsnorm_bwd(x: torch.Tensor, dy: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor) -> torch.Tensor:
    _require_cuda(x, dy, weight, rstd)
    x = _rows_operand(x)
    dy = _rows_operand(dy)
    w = weight.to(torch.bfloat16).contiguous()
    rows, D = x.shape
    dx = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    _check(_lib.vq_rmsnorm_bwd(x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), rows, D, w.data_ptr(),
                               rstd.contiguous().data_ptr(), dx.data_ptr(), dx.stride(0), _stream(x)))
    return dx


def add_rmsnorm_fwd(a: torch.Tensor, res: torch.Tensor, weight: torch.Tensor, eps: float):
    """(h = a + res, y = RMSNorm(h), rstd) for a, res [rows, D] bf16."""
    _require_cuda(a, res, weight)
    a = _rows_operand(a)
    res = _rows_operand(res)
    w = weight.to(torch.bfloat16).contiguous()
    rows, D = a.shape
    if res.shape != a.shape:
        raise ValueError(f"add_rmsnorm: shapes {tuple(a.shape)} and {tuple(res.shape)} differ")
    h = torch.empty(rows, D, dtype=torch.bfloat16, device=a.device)
    y = torch.empty(rows, D, dtype=torch.bfloat16, device=a.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=a.device)
    _check(_lib.vq_add_rmsnorm_fwd(a.data_ptr(), a.stride(0), res.data_ptr(), res.stride(0), rows, D, w.data_ptr(),
                                   float(eps), h.data_ptr(), h.stride(0), y.data_ptr(), y.stride(0), rstd.data_ptr(),
                                   _stream(a)))
    return h, y, rstd


def rmsnorm_bwd_add(x: torch.Tensor, dy: torch.Tensor, dres: torch.Tensor, weight: torch.Tensor,
                    rstd: torch.Tensor) -> torch.Tensor:
    """RMSNorm input gradient of dy at x, plus dres (fp32 sum, one rounding)."""
    _require_cuda(x, dy, dres, weight, rstd)
    x = _rows_operand(x)
    dy = _rows_operand(dy)
    dres = _rows_operand(dres)
    w = weight.to(torch.bfloat16).contiguous()
    rows, D = x.shape
    dx = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    _check(_lib.vq_rmsnorm_bwd_add(x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), dres.data_ptr(),
                                   dres.stride(0), rows, D, w.data_ptr(), rstd.contiguous().data_ptr(), dx.data_ptr(),
                                   dx.stride(0), _stream(x)))
    return dx


def _bshd(t: torch.Tensor) -> torch.Tensor:
    t = t.to(torch.bfloat16)
    if t.stride(-1) != 1 or any(st % 8 for st in t.stride()[:3]) or t.data_ptr() % 16 != 0:
        t = t.contiguous()
    return t


def rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, backward: bool = False):
    """Rotary embedding of q [B, S, Hq, D] and k [B, S, Hk, D] with cos/sin
    [B, S, D] (any strides with unit stride over D); returns contiguous
    [B, S, H, D] outputs (the transposed rotation when ``backward``)."""
    _require_cuda(q, k, cos, sin)
    q, k = _bshd(q), _bshd(k)
    B, S, Hq, D = q.shape
    Hk = k.shape[2]
    cos = cos.to(torch.bfloat16).expand(B, S, D)
    sin = sin.to(torch.bfloat16).expand(B, S, D)
    if cos.stride() != sin.stride() or cos.stride(-1) != 1 or cos.data_ptr() % 16 or sin.data_ptr() % 16 or \
            any(st % 8 for st in cos.stride()[:2]):
        cos, sin = cos.contiguous(), sin.contiguous()
    qo = torch.empty(B, S, Hq, D, dtype=torch.bfloat16, device=q.device)
    ko = torch.empty(B, S, Hk, D, dtype=torch.bfloat16, device=q.device)
    qs = (ctypes.c_int64 * 3)(q.stride(0), q.stride(1), q.stride(2))
    ks = (ctypes.c_int64 * 3)(k.stride(0), k.stride(1), k.stride(2))
    cs = (ctypes.c_int64 * 2)(cos.stride(0), cos.stride(1))
    _check(_lib.vq_rope(q.data_ptr(), qs, Hq, k.data_ptr(), ks, Hk, cos.data_ptr(), sin.data_ptr(), cs, B, S, D,
                        int(backward), qo.data_ptr(), ko.data_ptr(), _stream(q)))
    return qo, ko


def swiglu_fwd(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for [rows, F] operands."""
    _require_cuda(gate, up)
    gate, up = _rows_operand(gate), _rows_operand(up)
    rows, F = gate.shape
    y = torch.empty(rows, F, dtype=torch.bfloat16, device=gate.device)
    _check(_lib.vq_swiglu_fwd(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), rows, F, y.data_ptr(),
                              y.stride(0), _stream(gate)))
    return y


def swiglu_bwd(gate: torch.Tensor, up: torch.Tensor, dy: torch.Tensor, out: torch.Tensor | None = None):
    """(d gate, d up) of silu(gate) * up; with ``out`` ([rows, 2F] bf16,
    contiguous) both are written into it side by side and returned as views."""
    _require_cuda(gate, up, dy)
    gate, up, dy = _rows_operand(gate), _rows_operand(up), _rows_operand(dy)
    rows, F = gate.shape
    if out is not None:
        if out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, 2 * F) or not out.is_contiguous():
            raise ValueError("swiglu_bwd: out must be a contiguous bf16 [rows, 2F] tensor")
        dg, du = out[:, :F], out[:, F:]
    else:
        dg = torch.empty(rows, F, dtype=torch.bfloat16, device=gate.device)
        du = torch.empty(rows, F, dtype=torch.bfloat16, device=gate.device)
    _check(_lib.vq_swiglu_bwd(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0), dy.data_ptr(), dy.stride(0),
                              rows, F, dg.data_ptr(), du.data_ptr(), dg.stride(0), _stream(gate)))
    return dg, du



# ---------------------------------------------------------------- head norms with rotation
def _heads_operand(t: torch.Tensor):
    """(t, its strides over B, S, H): t copied where its strides over the others are no multiples of 8, that over D is
    not 1 or its first value is not 16-byte aligned."""
    b, s, h, d = t.stride()
    if d != 1 or (b | s | h) & 7 or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        b, s, h, d = t.stride()
    return t, b, s, h


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if not t.is_contiguous() or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _table_operand(t: torch.Tensor):
    """A rotary table with unit stride over R, the others multiples of 8, 16-byte aligned; copied otherwise."""
    st = t.stride()
    if st[-1] != 1 or st[-2] & 7 or (len(st) == 3 and st[0] & 7) or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _qk_operands(q, k, q_weight, k_weight, cos, sin):
    """Checked and laid out operands: device, q, k with their strides, weights, tables, (B, S, D, R), dtype code."""
    dev = _device_of(q, k, q_weight, k_weight, cos, sin)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[:2] != ks[:2] or qs[3] != ks[3]:
        raise ValueError(f"qk_norm_rope: q [B, S, Hq, D] and k [B, S, Hk, D] expected, got {tuple(qs)} and {tuple(ks)}")
    dt = q.dtype
    dtype = _float_code(q, "qk_norm_rope")
    if k.dtype != dt:
        raise ValueError(f"qk_norm_rope: q is {dt}, k is {k.dtype}")
    B, S, _, D = qs
    if q_weight.shape != (D,) or k_weight.shape != (D,):
        raise ValueError(f"qk_norm_rope: weights of shape ({D},) expected, got {tuple(q_weight.shape)} and "
                         f"{tuple(k_weight.shape)}")
    cshape = cos.shape
    if (len(cshape) not in (2, 3) or sin.shape != cshape or cshape[-2] != S
            or (len(cshape) == 3 and cshape[0] not in (1, B))):
        raise ValueError(f"qk_norm_rope: cos and sin [B or 1, S, R] expected, got {tuple(cshape)} and "
                         f"{tuple(sin.shape)} for q {tuple(qs)}")
    if q_weight.dtype != dt or k_weight.dtype != dt:
        _float_code(q_weight, "qk_norm_rope weight"), _float_code(k_weight, "qk_norm_rope weight")
        q_weight, k_weight = q_weight.float(), k_weight.float()
    if cos.dtype != dt or sin.dtype != dt:
        _float_code(cos, "qk_norm_rope table"), _float_code(sin, "qk_norm_rope table")
        cos, sin = cos.float(), sin.float()
    cos, sin = _table_operand(cos), _table_operand(sin)
    if cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    cst = cos.stride()
    cb = cst[0] if len(cshape) == 3 and cshape[0] > 1 else 0  # one table for every batch entry
    return (dev, _heads_operand(q), _heads_operand(k), _aligned(q_weight), _aligned(k_weight), cos, sin, cb, cst[-2],
            (B, S, D, cshape[-1]), dtype)


_strides3 = ctypes.c_int64 * 3
_CONTIGUOUS = torch.contiguous_format
_strides2 = ctypes.c_int64 * 2


def qk_norm_rope_fwd(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                     cos: torch.Tensor, sin: torch.Tensor, eps: float, weight_offset: float = 0.0, saved: bool = False):
    """Norm of each head of q [B, S, Hq, D] and k [B, S, Hk, D] (float32, bfloat16 or float16, any strides) with
    weights ``weight_offset + weight`` [D], then the rotation of its first R values by cos / sin [B or 1, S, R];
    contiguous outputs of q's type, rounded once.  ``saved``: also the operands as they were laid out, for
    ``qk_norm_rope_bwd``."""
    dev, (q, qb, qs, qh), (k, kb, ks, kh), wq, wk, c, s, cb, cs, (B, S, D, R), dtype = \
        _qk_operands(q, k, q_weight, k_weight, cos, sin)
    qo, ko = torch.empty_like(q, memory_format=_CONTIGUOUS), torch.empty_like(k, memory_format=_CONTIGUOUS)
    qst, kst, cst = _strides3(qb, qs, qh), _strides3(kb, ks, kh), _strides2(cb, cs)
    wf, cf = wq.dtype == torch.float32, c.dtype == torch.float32
    _check(_lib.vq_qk_norm_rope_fwd(q.data_ptr(), qst, q.shape[2], k.data_ptr(), kst, k.shape[2], wq.data_ptr(),
                                    wk.data_ptr(), wf, c.data_ptr(), s.data_ptr(), cst, cf, B, S, D, R, eps,
                                    weight_offset, dtype, qo.data_ptr(), ko.data_ptr(), _raw_stream(dev)))
    if saved:
        return qo, ko, (q, k, wq, wk, c, s), (dev, qst, kst, wf, cst, cf, B, S, D, R, eps, weight_offset, dtype)
    return qo, ko


def qk_norm_rope_bwd(gq: torch.Tensor, gk: torch.Tensor, operands, layout, want_weight_grads: bool = True):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope_fwd`` for the outputs' gradients gq, gk, from what it saved; the
    weights' gradients (in the type the weights were laid out in) are None unless wanted."""
    q, k, wq, wk, c, s = operands
    dev, qst, kst, wf, cst, cf, B, S, D, R, eps, weight_offset, dtype = layout
    if gq.shape != q.shape or gk.shape != k.shape or gq.dtype != q.dtype or gk.dtype != q.dtype:
        raise ValueError(f"qk_norm_rope: gradients of the outputs' shapes and type expected, got {tuple(gq.shape)} "
                         f"{gq.dtype} and {tuple(gk.shape)} {gk.dtype}")
    if gq.get_device() != dev or gk.get_device() != dev:
        raise ValueError("qk_norm_rope: gradients on the outputs' device expected")
    (gq, gqb, gqs, gqh), (gk, gkb, gks, gkh) = _heads_operand(gq), _heads_operand(gk)
    dq, dk = torch.empty_like(q, memory_format=_CONTIGUOUS), torch.empty_like(k, memory_format=_CONTIGUOUS)
    dwq = dwk = ws = None
    need = 0
    if want_weight_grads:
        dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
        need = _workspace_bytes("vq_qk_norm_rope_workspace_bytes", D)
        ws = q.new_empty(need, dtype=torch.uint8)
    _check(_lib.vq_qk_norm_rope_bwd(gq.data_ptr(), _strides3(gqb, gqs, gqh), gk.data_ptr(), _strides3(gkb, gks, gkh),
                                    q.data_ptr(), qst, q.shape[2], k.data_ptr(), kst, k.shape[2], wq.data_ptr(),
                                    wk.data_ptr(), wf, c.data_ptr(), s.data_ptr(), cst, cf, B, S, D, R, eps,
                                    weight_offset, dtype, dq.data_ptr(), dk.data_ptr(), _ptr(dwq), _ptr(dwk), _ptr(ws),
                                    need, _raw_stream(dev)))
    return dq, dk, dwq, dwk


# ---------------------------------------------------------------- gated embedding
def _ids_operand(ids: torch.Tensor) -> torch.Tensor:
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"token ids must be int64 or int32, got {ids.dtype}")
    return ids.contiguous()


class EmbedTable:
    """The checked packed candidates of an embedding table: what ``embed_mix`` and ``embed_gategrad`` pass on.  Holds
    the blocks; nothing of it outlives the call (or the backward) that made it."""

    __slots__ = ("blocks", "rows", "padded_cols", "cols", "device", "K", "types", "ptrs")

    def __init__(self, qtypes, qbytes, rows: int, padded_cols: int, cols: int):
        K = len(qtypes)
        if not 1 <= K <= 8 or K != len(qbytes):
            raise ValueError(f"1..8 candidates with their blocks expected, got {K} types and {len(qbytes)} tensors")
        if rows < 0 or cols < 0 or cols > padded_cols or padded_cols % 256:
            raise ValueError(f"table of {rows} rows: {padded_cols} stored columns must be a multiple of 256 that holds "
                             f"{cols}")
        self.device = _device_of(*qbytes)
        self.blocks, self.rows, self.padded_cols, self.cols, self.K = tuple(qbytes), rows, padded_cols, cols, K
        self.types, self.ptrs = (_int * K)(), (_vp * K)()
        for i, (qt, qb) in enumerate(zip(qtypes, qbytes)):
            be, bb = _geometry(qt)
            if qb.dtype != torch.uint8 or not qb.is_contiguous() or qb.numel() != rows * (padded_cols // be) * bb:
                raise ValueError(f"{qt}: contiguous uint8 blocks of {rows * (padded_cols // be) * bb} bytes expected, got "
                                 f"{qb.dtype} {tuple(qb.shape)}")
            self.types[i] = GGML_TYPE[qt]
            self.ptrs[i] = qb.data_ptr()

    def check(self, *ts: torch.Tensor) -> None:
        for t in ts:
            if t.get_device() != self.device:
                _require_cuda(*ts)
                raise ValueError(f"tensors on cuda:{self.device} expected, got {t.device}")

    def check_plan(self, plan: torch.Tensor) -> None:
        self.check(plan)
        if plan.dtype != torch.uint8 or not plan.is_contiguous():
            raise ValueError(f"a plan as embed_plan made it expected, got {plan.dtype} {tuple(plan.shape)} with strides "
                             f"{plan.stride()}")


def embed_plan(ids: torch.Tensor, rows: int, vocab_start: int | None = None) -> torch.Tensor:
    """Plan of the token ids over a table of ``rows`` rows (uint8, its layout is the C header's): the tokens sorted by
    row and cut into pieces of equal rows, for ``embed_mix`` and ``embed_gategrad`` of the same ids and table."""
    dev = _device_of(ids)
    ids = _ids_operand(ids)
    T = ids.numel()
    need = _lib.vq_embed_plan_bytes(T)
    plan = torch.empty(need, dtype=torch.uint8, device=ids.device)
    _check(_lib.vq_embed_plan(ids.data_ptr(), ids.dtype == torch.int32, T, vocab_start or 0, rows, plan.data_ptr(),
                              need, _raw_stream(dev)))
    return plan


def embed_mix(ids: torch.Tensor, table: EmbedTable, probs: torch.Tensor, scale: float = 1.0,
              vocab_start: int | None = None, plan: torch.Tensor | None = None) -> torch.Tensor:
    """Rows scale * sum_k probs[k] W_k[ids] of a table of packed candidates -> bf16 [*ids.shape, cols].  With
    ``vocab_start`` the table holds the vocabulary from there on and tokens of other shards get rows of zeros;
    without it such ids are reported by ``device_error`` as well.  With the ids' ``plan`` a row is decoded once for
    up to 8 tokens that name it, else once per token."""
    table.check(ids, probs)
    ids = _ids_operand(ids)
    if plan is not None:
        table.check_plan(plan)
    if probs.numel() != table.K:
        raise ValueError(f"{table.K} probabilities expected, got {tuple(probs.shape)}")
    if probs.dtype != torch.float32 or not probs.is_contiguous():
        probs = probs.detach().to(torch.float32).contiguous()
    cols = table.cols
    out = torch.empty(*ids.shape, cols, dtype=torch.bfloat16, device=ids.device)
    _check(_lib.vq_embed_mix(table.K, table.types, table.ptrs, probs.data_ptr(), ids.data_ptr(), ids.dtype == torch.int32,
                             ids.numel(), _ptr(plan), 0 if plan is None else plan.numel(), vocab_start or 0, table.rows,
                             table.padded_cols, cols, scale, vocab_start is None, out.data_ptr(), cols,
                             _raw_stream(table.device)))
    return out


def embed_gategrad(dy: torch.Tensor, table: EmbedTable, plan: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """grad[k] = scale * sum_t <dy[t], W_k[ids[t]]> (float32 [K]) for dy [..., cols] in float32, bfloat16 or float16 and
    the plan of its ids; ids outside the table add nothing."""
    table.check(dy)
    table.check_plan(plan)
    K, cols = table.K, table.cols
    code = _float_code(dy, "embed_gategrad")
    if dy.dim() < 1 or dy.shape[-1] != cols:
        raise ValueError(f"gradient rows of {cols} columns expected, got {tuple(dy.shape)}")
    if dy.dim() != 2:
        dy = dy.reshape(-1, cols) if cols else dy.new_empty(0, 0)
    T = dy.shape[0]
    nplan = plan.numel()
    ld, unit = dy.stride()
    if unit != 1 or ld < cols:
        dy, ld = dy.contiguous(), cols
    need = _workspace_bytes("vq_embed_gategrad_workspace_bytes", K)
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device)
    g = torch.empty(K, dtype=torch.float32, device=dy.device)
    _check(_lib.vq_embed_gategrad(K, table.types, table.ptrs, plan.data_ptr(), nplan, T, table.rows, table.padded_cols,
                                  cols, scale, dy.data_ptr(), ld, code, ws.data_ptr(), need, g.data_ptr(),
                                  _raw_stream(table.device)))
    return g


# ---------------------------------------------------------------- global norm and clipping
_dtype_of, _nbytes_of = attrgetter("dtype"), attrgetter("nbytes")


class NotContiguous(ValueError):
    """A tensor is sparse or has strides of its own."""


def clip_grad_norm(tensors, max_norm: float = float("inf"), norm_inf: bool = False) -> torch.Tensor:
    """Global 2-norm (or largest magnitude) of dense, non-overlapping CUDA tensors as a float32 scalar on their device,
    and every value times min(1, max_norm / (norm + 1e-6)) in place; an infinite ``max_norm`` leaves them as they are."""
    n = len(tensors)
    if n == 0:
        raise ValueError("clip_grad_norm: no tensors")
    no_tangents("clip_grad_norm", tensors)
    # one pass per property: a few hundred short tensors cost more here than on the GPU
    dev = _device_of(tensors[0])
    if set(map(torch.Tensor.get_device, tensors)) != {dev}:
        _device_of(*tensors)
    if not all(map(torch.Tensor.is_contiguous, tensors)):  # nor is a sparse one
        raise NotContiguous("clip_grad_norm: contiguous tensors expected")
    types = set(map(_dtype_of, tensors))
    for d in types:
        if d not in _FLOAT_CODE:
            raise ValueError(f"clip_grad_norm: float32, bfloat16 or float16 expected, got {d}")
    codes = array("i", [_FLOAT_CODE[types.pop()]]) * n if len(types) == 1 else \
        array("i", [_FLOAT_CODE[t.dtype] for t in tensors])
    ptrs = array("Q", map(torch.Tensor.data_ptr, tensors))
    sizes = array("q", map(_nbytes_of, tensors))
    if max_norm != math.inf:  # a graph that has saved one of them must notice
        torch.autograd.graph.increment_version(tensors)
    device = tensors[0].device
    norm = torch.empty((), dtype=torch.float32, device=device)
    need = _lib.vq_clip_grad_norm_workspace_bytes(n)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _check(_lib.vq_clip_grad_norm(n, ptrs.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], max_norm,
                                  norm_inf, ws.data_ptr(), need, norm.data_ptr(), _raw_stream(dev)))
    return norm
