"""Python binding of libcuflash_attn.so (MI355X / gfx950).

Mirrors the reference's ctypes caller (tests/integration/test_pytorch_comparison.py:37-194 and
examples/python_binding.py:51-180): the same library search order ($CUFLASH_LIB, then
build/libcuflash_attn.so and the build/<preset>/ directories), the same argtypes for the six
C-ABI entry points, and status codes equal to cuflash::FlashAttentionError. On top of that it
offers tensor-level helpers for PyTorch-ROCm tensors that allocate the outputs and enqueue on
torch's current HIP stream.

There is no fallback: if the library is missing, load_library() raises.
"""

from __future__ import annotations

import ctypes
import os
import sys
from typing import Optional, Sequence

SUCCESS = 0
INVALID_DIMENSION = 1
DIMENSION_MISMATCH = 2
NULL_POINTER = 3
CUDA_ERROR = 4
OUT_OF_MEMORY = 5
UNSUPPORTED_HEAD_DIM = 6
UNSUPPORTED_DTYPE = 7

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(os.path.dirname(_PKG_DIR))

_DTYPE_SUFFIX = {"float32": "f32", "float16": "f16", "bfloat16": "bf16"}


class CuFlashError(RuntimeError):
    """Raised by the tensor helpers when a C-ABI call returns a non-zero status."""

    def __init__(self, code: int, message: str):
        super().__init__(f"cuflash error {code}: {message}")
        self.code = code


def candidate_library_paths() -> Sequence[str]:
    """Search order of the reference's test_pytorch_comparison.py:158-180."""
    build_dir = os.path.join(REPO_ROOT, "build")
    out = []
    explicit = os.environ.get("CUFLASH_LIB")
    if explicit:
        out.append(explicit)
    name = "libcuflash_attn.so"
    out.append(os.path.join(build_dir, name))
    for preset in ("default", "release", "release-fast-math", "minimal", "Release", "Debug"):
        out.append(os.path.join(build_dir, preset, name))
    return out


_FWD_ARGS = [ctypes.c_void_p] * 5 + [ctypes.c_int] * 4 + [ctypes.c_float, ctypes.c_bool,
                                                          ctypes.c_void_p]
_BWD_ARGS = [ctypes.c_void_p] * 9 + [ctypes.c_int] * 4 + [ctypes.c_float, ctypes.c_bool,
                                                          ctypes.c_void_p]
_DEC_ARGS = [ctypes.c_void_p] * 5 + [ctypes.c_int] * 4 + [ctypes.c_float, ctypes.c_int,
                                                          ctypes.c_void_p]
_DEC_GQA_ARGS = [ctypes.c_void_p] * 5 + [ctypes.c_int] * 5 + [ctypes.c_float, ctypes.c_int,
                                                              ctypes.c_void_p]
_DEC_PAGED_ARGS = [ctypes.c_void_p] * 7 + [ctypes.c_int] * 6 + [ctypes.c_float, ctypes.c_int,
                                                                ctypes.c_void_p]
_FWD_EXT_ARGS = [ctypes.c_void_p] * 5 + [ctypes.c_int] * 6 + [ctypes.c_float, ctypes.c_bool,
                                                              ctypes.c_void_p]
_BWD_EXT_ARGS = [ctypes.c_void_p] * 9 + [ctypes.c_int] * 6 + [ctypes.c_float, ctypes.c_bool,
                                                              ctypes.c_void_p]

_APPEND_PAGED_ARGS = ([ctypes.c_void_p] * 11 + [ctypes.c_int] * 13 +
                      [ctypes.c_bool, ctypes.c_void_p])
_FWD_PAGED_ARGS = ([ctypes.c_void_p] * 8 + [ctypes.c_int] * 7 +
                   [ctypes.c_float, ctypes.c_bool, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p])
_DEC_SHARED_ARGS = ([ctypes.c_void_p] * 8 + [ctypes.c_int] * 7 +
                    [ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p])

_APPEND_PAGED_Q8_ARGS = ([ctypes.c_void_p] * 13 + [ctypes.c_int] * 13 +
                         [ctypes.c_bool, ctypes.c_int, ctypes.c_void_p])
_READ_PAGED_Q8_ARGS = [ctypes.c_void_p] * 9 + [ctypes.c_int] * 8 + [ctypes.c_void_p]
_DEC_PAGED_Q8_ARGS = ([ctypes.c_void_p] * 9 + [ctypes.c_int] * 6 +
                      [ctypes.c_float, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t,
                       ctypes.c_void_p])
_FWD_PAGED_Q8_ARGS = ([ctypes.c_void_p] * 10 + [ctypes.c_int] * 7 +
                      [ctypes.c_float, ctypes.c_bool, ctypes.c_int, ctypes.c_void_p,
                       ctypes.c_size_t, ctypes.c_void_p])

EXPORTED_SYMBOLS = (
    "cuflash_attention_forward_f32", "cuflash_attention_forward_f16",
    "cuflash_attention_forward_bf16", "cuflash_attention_backward_f32",
    "cuflash_attention_backward_f16", "cuflash_attention_backward_bf16",
    "cuflash_attention_decode_f32", "cuflash_attention_decode_f16",
    "cuflash_attention_decode_bf16", "cuflash_attention_decode_gqa_f32",
    "cuflash_attention_decode_gqa_f16", "cuflash_attention_decode_gqa_bf16",
    "cuflash_attention_decode_paged_f32", "cuflash_attention_decode_paged_f16",
    "cuflash_attention_decode_paged_bf16", "cuflash_attention_forward_ext_f32",
    "cuflash_attention_forward_ext_f16", "cuflash_attention_forward_ext_bf16",
    "cuflash_attention_backward_ext_f32", "cuflash_attention_backward_ext_f16",
    "cuflash_attention_backward_ext_bf16", "cuflash_error_string", "cuflash_version",
    "cuflash_profile_enable", "cuflash_profile_report", "cuflash_attention_decode_noalloc_f16",
    "cuflash_release_workspaces",
)

# Declared in include/cuflash/paged_cache.h.
PAGED_CACHE_SYMBOLS = tuple(f"cuflash_attention_{kind}_{sfx}"
                            for kind in ("append_paged", "forward_paged", "decode_shared",
                                         "forward_paged_workspace", "decode_shared_workspace")
                            for sfx in ("f32", "f16", "bf16"))


# Declared in include/cuflash/paged_cache_q8.h.
PAGED_CACHE_Q8_SYMBOLS = tuple(f"cuflash_attention_{kind}_{sfx}"
                               for kind in ("append_paged_q8", "read_paged_q8", "decode_paged_q8",
                                            "forward_paged_q8", "decode_paged_q8_workspace",
                                            "forward_paged_q8_workspace")
                               for sfx in ("f32", "f16", "bf16"))


class CuFlashLibrary:
    """ctypes view of libcuflash_attn.so with argtypes set (reference CuFlashLibrary)."""

    def __init__(self, library: ctypes.CDLL):
        self.library = library
        self.path = getattr(library, "_name", "")
        for sfx in ("f32", "f16", "bf16"):
            fwd = getattr(library, f"cuflash_attention_forward_{sfx}")
            fwd.argtypes, fwd.restype = _FWD_ARGS, ctypes.c_int
            bwd = getattr(library, f"cuflash_attention_backward_{sfx}")
            bwd.argtypes, bwd.restype = _BWD_ARGS, ctypes.c_int
            dec = getattr(library, f"cuflash_attention_decode_{sfx}")
            dec.argtypes, dec.restype = _DEC_ARGS, ctypes.c_int
            gqa = getattr(library, f"cuflash_attention_decode_gqa_{sfx}")
            gqa.argtypes, gqa.restype = _DEC_GQA_ARGS, ctypes.c_int
            paged = getattr(library, f"cuflash_attention_decode_paged_{sfx}")
            paged.argtypes, paged.restype = _DEC_PAGED_ARGS, ctypes.c_int
            fwd_ext = getattr(library, f"cuflash_attention_forward_ext_{sfx}")
            fwd_ext.argtypes, fwd_ext.restype = _FWD_EXT_ARGS, ctypes.c_int
            bwd_ext = getattr(library, f"cuflash_attention_backward_ext_{sfx}")
            bwd_ext.argtypes, bwd_ext.restype = _BWD_EXT_ARGS, ctypes.c_int
            append = getattr(library, f"cuflash_attention_append_paged_{sfx}")
            append.argtypes, append.restype = _APPEND_PAGED_ARGS, ctypes.c_int
            fwd_paged = getattr(library, f"cuflash_attention_forward_paged_{sfx}")
            fwd_paged.argtypes, fwd_paged.restype = _FWD_PAGED_ARGS, ctypes.c_int
            shared = getattr(library, f"cuflash_attention_decode_shared_{sfx}")
            shared.argtypes, shared.restype = _DEC_SHARED_ARGS, ctypes.c_int
            for kind, n in (("forward_paged", 5), ("decode_shared", 4)):
                size = getattr(library, f"cuflash_attention_{kind}_workspace_{sfx}")
                size.argtypes, size.restype = [ctypes.c_int] * n, ctypes.c_longlong
            for kind, args in (("append_paged_q8", _APPEND_PAGED_Q8_ARGS),
                               ("read_paged_q8", _READ_PAGED_Q8_ARGS),
                               ("decode_paged_q8", _DEC_PAGED_Q8_ARGS),
                               ("forward_paged_q8", _FWD_PAGED_Q8_ARGS)):
                q8 = getattr(library, f"cuflash_attention_{kind}_{sfx}")
                q8.argtypes, q8.restype = args, ctypes.c_int
            for kind, n in (("forward_paged_q8", 5), ("decode_paged_q8", 4)):
                size = getattr(library, f"cuflash_attention_{kind}_workspace_{sfx}")
                size.argtypes, size.restype = [ctypes.c_int] * n, ctypes.c_longlong
        noalloc = library.cuflash_attention_decode_noalloc_f16
        noalloc.argtypes, noalloc.restype = _DEC_ARGS, ctypes.c_int
        library.cuflash_error_string.argtypes = [ctypes.c_int]
        library.cuflash_error_string.restype = ctypes.c_char_p
        library.cuflash_version.argtypes = []
        library.cuflash_version.restype = ctypes.c_char_p
        library.cuflash_profile_enable.argtypes = [ctypes.c_int]
        library.cuflash_profile_enable.restype = None
        library.cuflash_profile_report.argtypes = [ctypes.c_char_p, ctypes.c_int]
        library.cuflash_profile_report.restype = ctypes.c_int
        library.cuflash_release_workspaces.argtypes = []
        library.cuflash_release_workspaces.restype = ctypes.c_int

    def error_string(self, code: int) -> str:
        return self.library.cuflash_error_string(int(code)).decode()

    def version(self) -> str:
        return self.library.cuflash_version().decode()

    def profile_enable(self, enabled: bool) -> None:
        self.library.cuflash_profile_enable(1 if enabled else 0)

    def profile_report(self) -> dict:
        """{label: (launches, total_ms)} for the kernels launched since the last report."""
        buf = ctypes.create_string_buffer(1 << 16)
        self.library.cuflash_profile_report(buf, len(buf))
        out = {}
        for line in buf.value.decode().splitlines():
            label, count, ms = line.split("\t")
            out[label] = (int(count), float(ms))
        return out

    def fn(self, kind: str, suffix: str):
        return getattr(self.library, f"cuflash_attention_{kind}_{suffix}")


_CACHED: Optional[CuFlashLibrary] = None


def load_library(path: Optional[str] = None) -> CuFlashLibrary:
    """Loads libcuflash_attn.so (first hit of the search order). Raises when it is missing."""
    global _CACHED
    if path is None and _CACHED is not None:
        return _CACHED
    tried = [path] if path else list(candidate_library_paths())
    errors = []
    for p in tried:
        if not os.path.exists(p):
            errors.append(f"{p}: missing")
            continue
        try:
            lib = CuFlashLibrary(ctypes.CDLL(p))
        except OSError as e:
            errors.append(f"{p}: {e}")
            continue
        if path is None:
            _CACHED = lib
        return lib
    raise OSError("libcuflash_attn.so not found; build it with "
                  "`python cuflash-attn_amd/build.py`. Tried:\n  " + "\n  ".join(errors))


# ---------------------------------------------------------------------------------------------
# PyTorch tensor helpers (device memory and streams come from PyTorch-ROCm)
# ---------------------------------------------------------------------------------------------

_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch  # noqa: WPS433 (imported lazily: the ctypes layer itself needs no torch)

        _TORCH = torch
    return _TORCH


def _suffix(t) -> str:
    name = str(t.dtype).replace("torch.", "")
    if name not in _DTYPE_SUFFIX:
        raise CuFlashError(UNSUPPORTED_DTYPE, f"unsupported dtype {t.dtype}")
    return _DTYPE_SUFFIX[name]


def _check(tensors, dtype):
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("tensors must be on the GPU")
        if not t.is_contiguous():
            raise ValueError("tensors must be contiguous")
        if t.dtype != dtype:
            raise ValueError("all tensors must share one dtype")


def _stream_ptr(stream=None):
    if stream is not None:
        return stream.cuda_stream
    # The handle of torch.cuda.current_stream() without building a Stream object around it (2.8 us
    # of a small call's 12.8), where this torch has the internal function for it.
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None:
        return torch.cuda.current_stream().cuda_stream
    return raw(torch.cuda.current_device())


def _raise(lib: CuFlashLibrary, status: int):
    if status != SUCCESS:
        raise CuFlashError(status, lib.error_string(status))


def flash_attention_forward(q, k, v, scale: Optional[float] = None, causal: bool = False,
                            out=None, lse=None, stream=None, lib: Optional[CuFlashLibrary] = None):
    """O, L = attention(q, k, v) for [B, H, N, D] tensors; L is float32 [B, H, N]."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k, v), q.dtype)
    B, H, N, D = q.shape
    if k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must have the same shape")
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = torch.empty_like(q) if out is None else out
    lse = q.new_empty((B, H, N), dtype=torch.float32) if lse is None else lse
    status = lib.fn("forward", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                           out.data_ptr(), lse.data_ptr(), B, H, N, D, scale,
                                           bool(causal), _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


def flash_attention_backward(q, k, v, o, lse, do, scale: Optional[float] = None,
                             causal: bool = False, stream=None,
                             lib: Optional[CuFlashLibrary] = None):
    """dQ, dK, dV for [B, H, N, D] tensors given O and the float32 logsumexp L."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k, v, o, do), q.dtype)
    B, H, N, D = q.shape
    scale = float(D ** -0.5) if scale is None else float(scale)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    status = lib.fn("backward", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                            o.data_ptr(), lse.data_ptr(), do.data_ptr(),
                                            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, H, N,
                                            D, scale, bool(causal), _stream_ptr(stream))
    _raise(lib, status)
    return dq, dk, dv


def _ext_shapes(q, k, v):
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError("expected q [B,H,Nq,D] and k, v [B,Hkv,Nk,D]")
    B, H, Nq, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError("q and k, v differ in batch or head_dim")
    return B, H, k.shape[1], Nq, k.shape[2], D


def flash_attention_forward_ext(q, k, v, scale: Optional[float] = None, causal: bool = False,
                                out=None, lse=None, stream=None,
                                lib: Optional[CuFlashLibrary] = None):
    """Forward with q [B, H, Nq, D] and k, v [B, Hkv, Nk, D] (Hkv a divisor of H; query head h
    reads key/value head h // (H // Hkv)), D in {32, 64, 96, 128, 256}; a causal mask lets
    query i see keys j <= i + Nk - Nq (cuflash_attention_forward_ext_*).
    -> O [B, H, Nq, D], L float32 [B, H, Nq]."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k, v), q.dtype)
    B, H, Hkv, Nq, Nk, D = _ext_shapes(q, k, v)
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = torch.empty_like(q) if out is None else out
    lse = q.new_empty((B, H, Nq), dtype=torch.float32) if lse is None else lse
    status = lib.fn("forward_ext", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                               out.data_ptr(), lse.data_ptr(), B, H, Hkv, Nq,
                                               Nk, D, scale, bool(causal), _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


def flash_attention_backward_ext(q, k, v, o, lse, do, scale: Optional[float] = None,
                                 causal: bool = False, stream=None,
                                 lib: Optional[CuFlashLibrary] = None):
    """dQ [B, H, Nq, D], dK, dV [B, Hkv, Nk, D] for the shapes of flash_attention_forward_ext
    (dK, dV of a key/value head summed over its query heads; cuflash_attention_backward_ext_*)."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k, v, o, do), q.dtype)
    B, H, Hkv, Nq, Nk, D = _ext_shapes(q, k, v)
    scale = float(D ** -0.5) if scale is None else float(scale)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    status = lib.fn("backward_ext", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                o.data_ptr(), lse.data_ptr(), do.data_ptr(),
                                                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, H,
                                                Hkv, Nq, Nk, D, scale, bool(causal),
                                                _stream_ptr(stream))
    _raise(lib, status)
    return dq, dk, dv


def flash_attention_decode(q, k, v, scale: Optional[float] = None, num_splits: int = 0,
                           out=None, lse=None, stream=None,
                           lib: Optional[CuFlashLibrary] = None):
    """Split-KV decode: q [B, H, 1, D], k/v [B, Hkv, Lkv, D] -> O [B, H, 1, D], L [B, H, 1].
    Hkv == H calls cuflash_attention_decode_*, a divisor of H (grouped-query / multi-query
    attention: query head h reads key/value head h // (H // Hkv)) cuflash_attention_decode_gqa_*."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k, v), q.dtype)
    B, H, one, D = q.shape
    if one != 1 or k.dim() != 4 or k.shape[0] != B or k.shape[3] != D or v.shape != k.shape:
        raise ValueError("decode expects q [B,H,1,D] and k, v [B,Hkv,Lkv,D]")
    Hkv, kv_len = k.shape[1], k.shape[2]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = torch.empty_like(q) if out is None else out
    lse = q.new_empty((B, H, 1), dtype=torch.float32) if lse is None else lse
    if Hkv == H:
        status = lib.fn("decode", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                              out.data_ptr(), lse.data_ptr(), B, H, kv_len, D,
                                              scale, int(num_splits), _stream_ptr(stream))
    else:
        status = lib.fn("decode_gqa", _suffix(q))(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                  out.data_ptr(), lse.data_ptr(), B, H, Hkv,
                                                  kv_len, D, scale, int(num_splits),
                                                  _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


def flash_attention_decode_paged(q, k_cache, v_cache, block_table, seq_lens,
                                 scale: Optional[float] = None, num_splits: int = 0, out=None,
                                 lse=None, stream=None, lib: Optional[CuFlashLibrary] = None):
    """Split-KV decode over a paged cache: q [B, H, 1, D]; k_cache, v_cache
    [num_pages, page_size, Hkv, D]; block_table [B, max_pages] int32 (page of keys
    [p * page_size, (p + 1) * page_size) of each sequence); seq_lens [B] int32.
    -> O [B, H, 1, D], L [B, H, 1] (cuflash_attention_decode_paged_*)."""
    torch = _torch()
    lib = lib or load_library()
    _check((q, k_cache, v_cache), q.dtype)
    B, H, one, D = q.shape
    if (one != 1 or k_cache.dim() != 4 or k_cache.shape[3] != D or v_cache.shape != k_cache.shape
            or block_table.dim() != 2 or block_table.shape[0] != B
            or tuple(seq_lens.shape) != (B,)):
        raise ValueError("paged decode expects q [B,H,1,D], k/v cache [P,page,Hkv,D], "
                         "block_table [B,max_pages], seq_lens [B]")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_table and seq_lens must be int32")
    if not (block_table.is_contiguous() and seq_lens.is_contiguous()):
        raise ValueError("block_table and seq_lens must be contiguous")
    page_size, Hkv = k_cache.shape[1], k_cache.shape[2]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = torch.empty_like(q) if out is None else out
    lse = q.new_empty((B, H, 1), dtype=torch.float32) if lse is None else lse
    status = lib.fn("decode_paged", _suffix(q))(q.data_ptr(), k_cache.data_ptr(),
                                                v_cache.data_ptr(), out.data_ptr(),
                                                lse.data_ptr(), block_table.data_ptr(),
                                                seq_lens.data_ptr(), B, H, Hkv, page_size,
                                                block_table.shape[1], D, scale, int(num_splits),
                                                _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


def _check_paged(tensors, k_cache, v_cache, block_table, seq_lens, query_starts=None):
    """What the calls on a paged cache have in common: one device, the current one; K and V cache
    [P, page, Hkv, D] and contiguous; int32 tables. -> device, B, pages, page size, Hkv, D.
    Small calls wait for the host, so what is right is passed in one look at each tensor
    (2 us for eight of them); which rule is broken is found out afterwards."""
    torch = _torch()
    device = torch.cuda.current_device()
    dtype, int32 = k_cache.dtype, torch.int32
    ints = ((block_table, seq_lens) if query_starts is None
            else (block_table, seq_lens, query_starts))
    good = k_cache.is_contiguous() and v_cache.is_contiguous()
    for t in (k_cache, v_cache, *tensors):
        if t.get_device() != device or t.dtype is not dtype or t.data_ptr() & 15:
            good = False
    for t in ints:
        if t.get_device() != device or t.dtype is not int32 or not t.is_contiguous():
            good = False
    if not good:
        _refuse_paged(tensors, k_cache, v_cache, ints, device)
    shape, B = k_cache.shape, block_table.shape[0]
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("expected k_cache, v_cache [P,page,Hkv,D]")
    if block_table.dim() != 2 or seq_lens.shape != (B,):
        raise ValueError("expected block_table [B,max_pages] and seq_lens [B]")
    if query_starts is not None and query_starts.shape != (B + 1,):
        raise ValueError("expected query_starts [B+1]")
    return (device, B, *shape)


def _refuse_paged(tensors, k_cache, v_cache, ints, device):
    torch = _torch()
    _suffix(k_cache)
    every = (*tensors, k_cache, v_cache, *ints)
    if not all(t.is_cuda for t in every):
        raise ValueError("tensors must be on the GPU")
    if any(t.device.index != device for t in every):
        raise ValueError("tensors must be on the current device")
    if any(t.dtype != k_cache.dtype for t in (*tensors, v_cache)):
        raise ValueError("all tensors must share one dtype")
    if any(t.dtype != torch.int32 for t in ints):
        raise TypeError("block_table, seq_lens and query_starts must be int32")
    if not all(t.is_contiguous() for t in (k_cache, v_cache, *ints)):
        raise ValueError("the caches and int32 tensors must be contiguous")
    if any(t.data_ptr() % 16 for t in (*tensors, k_cache, v_cache)):
        raise ValueError("tensors must start at a multiple of 16 bytes")


def _output(given, like, shape, dtype, stream, name):
    """The caller's output, checked, or a new one that belongs to the call's stream."""
    if given is not None:
        if (tuple(given.shape) != tuple(shape) or given.dtype != dtype
                or given.device != like.device or not given.is_contiguous()
                or given.data_ptr() % 16):
            raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on the "
                             "inputs' device")
        return given
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _capturing(stream):
    """Whether the call's stream, torch's current one where that is None, is being captured."""
    torch = _torch()
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _captured_workspace(lib, kind, like, stream, *sizes):
    """Pointer and bytes of the workspace of a call that is being captured: torch's allocator gives it
    from the graph's own pool. Eager calls use the library's: None, 0. The third value keeps it."""
    torch = _torch()
    if not _capturing(stream):
        return None, 0, None
    need = lib.fn(f"{kind}_workspace", _suffix(like))(*sizes)
    if need <= 0:
        return None, 0, None
    ws = _output(None, like, (need,), torch.uint8, stream, "workspace")
    return ws.data_ptr(), need, ws


def _token_stride(x, name):
    """Elements from token to token of x [T, heads, D], whose heads lie side by side."""
    T, heads, D = x.shape
    apart, head, one = x.stride()
    if one != 1 or (heads > 1 and head != D):
        raise ValueError(f"the heads of a token of {name} must be contiguous")
    if T == 1:
        return heads * D
    if apart < heads * D or apart > 0x7fffffff or apart * x.element_size() % 16:
        raise ValueError(f"the tokens of {name} must be a multiple of 16 bytes apart, less than 2^31 "
                         "elements, and not overlap")
    return apart


def _rotation(cos, sin, device):
    """Positions and rotated elements of the tables of an append, checked; 0, 0 without."""
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is None:
        return 0, 0
    if cos.dim() != 2 or sin.shape != cos.shape:
        raise ValueError("expected cos, sin [positions, R / 2]")
    for x in (cos, sin):
        if x.dtype is not _torch().float32 or x.get_device() != device \
                or not x.is_contiguous() or x.data_ptr() & 15:
            raise ValueError("cos and sin must be contiguous float32 tensors on the inputs' "
                             "device")
    return cos.shape[0], 2 * cos.shape[1]


def flash_attention_append_paged(k, v, k_cache, v_cache, block_table, seq_lens,
                                 query_starts=None, q=None, cos=None, sin=None,
                                 interleaved: bool = False, out=None, stream=None,
                                 lib: Optional[CuFlashLibrary] = None):
    """Writes new tokens' k, v [T, Hkv, D] to the pages of their positions in k_cache, v_cache
    [P, page, Hkv, D] and rotates k, and q [T, H, D] if given, on the way (the tensors' tokens may
    lie apart, as in a projection's joint output). Tokens query_starts[b] .. query_starts[b + 1] - 1
    are the newest of sequence b, whose length with them is seq_lens[b]; without query_starts
    there is one token per sequence. cos, sin float32 [positions, R / 2]: the first R elements of a
    head are rotated, pairs (i, i + R / 2) or (2 i, 2 i + 1) if `interleaved`.
    -> rotated q [T, H, D] or None (cuflash_attention_append_paged_*)."""
    torch = _torch()
    lib = lib or load_library()
    given = (k, v) if q is None else (k, v, q)
    device, B, pages, page_size, Hkv, D = _check_paged(given, k_cache, v_cache, block_table,
                                                       seq_lens, query_starts)
    T = k.shape[0]
    H = 0 if q is None else q.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != (T, Hkv, D) \
            or (q is not None and q.shape != (T, H, D)):
        raise ValueError("expected k, v [T,Hkv,D] and q [T,H,D] of the cache's Hkv and D")
    positions, R = _rotation(cos, sin, device)
    k_stride, v_stride, q_stride = _token_stride(k, "k"), _token_stride(v, "v"), 0
    if q is not None:
        q_stride = _token_stride(q, "q")
        out = _output(out, q, (T, H, D), q.dtype, stream, "out")
    elif out is not None:
        raise ValueError("out is the rotated q: it needs q")
    q_ptr, out_ptr = (None, None) if q is None else (q.data_ptr(), out.data_ptr())
    cos_ptr, sin_ptr = (None, None) if cos is None else (cos.data_ptr(), sin.data_ptr())
    status = lib.fn("append_paged", _suffix(k))(
        q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, k_cache.data_ptr(), v_cache.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(),
        None if query_starts is None else query_starts.data_ptr(), cos_ptr, sin_ptr, T, B, H, Hkv,
        q_stride, k_stride, v_stride, pages, page_size, block_table.shape[1], D, R, positions,
        bool(interleaved), _stream_ptr(stream))
    _raise(lib, status)
    return out


def flash_attention_forward_paged(q, k_cache, v_cache, block_table, seq_lens, query_starts,
                                  scale: Optional[float] = None, causal: bool = False, out=None,
                                  lse=None, stream=None, lib: Optional[CuFlashLibrary] = None):
    """Attention of new tokens over a paged cache: q [T, H, D], tokens query_starts[b] ..
    query_starts[b + 1] - 1 being the newest of sequence b, whose keys, theirs among them, number
    seq_lens[b] (flash_attention_append_paged writes them). With `causal` a token sees the keys up
    to its own. Cache and block table as in flash_attention_decode_paged.
    -> O [T, H, D], L float32 [T, H] (cuflash_attention_forward_paged_*)."""
    torch = _torch()
    lib = lib or load_library()
    _, B, _, page_size, Hkv, D = _check_paged((q,), k_cache, v_cache, block_table, seq_lens,
                                              query_starts)
    if q.dim() != 3 or q.shape[2] != D or not q.is_contiguous():
        raise ValueError("expected contiguous q [T,H,D] of the cache's D")
    T, H = q.shape[:2]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = _output(out, q, (T, H, D), q.dtype, stream, "out")
    lse = _output(lse, q, (T, H), torch.float32, stream, "lse")
    ws, ws_bytes, _keep = _captured_workspace(lib, "forward_paged", q, stream, T, B, H, Hkv, D)
    status = lib.fn("forward_paged", _suffix(q))(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(), query_starts.data_ptr(), T, B, H, Hkv,
        page_size, block_table.shape[1], D, scale, bool(causal), ws, ws_bytes,
        _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


def flash_attention_decode_shared(q, k_cache, v_cache, prefix_table, prefix_len: int, block_table,
                                  seq_lens, scale: Optional[float] = None, out=None, lse=None,
                                  stream=None, lib: Optional[CuFlashLibrary] = None):
    """flash_attention_decode_paged for a batch whose first prefix_len keys are the same: they come
    from the pages of prefix_table [pages] int32 and are read once for the batch, the keys from
    prefix_len on from block_table (whose earlier entries are not used). seq_lens counts both.
    -> O [B, H, 1, D], L [B, H, 1] (cuflash_attention_decode_shared_*)."""
    torch = _torch()
    lib = lib or load_library()
    device, B, _, page_size, Hkv, D = _check_paged((q,), k_cache, v_cache, block_table, seq_lens)
    if q.dim() != 4 or q.shape[0] != B or q.shape[2] != 1 or q.shape[3] != D \
            or not q.is_contiguous():
        raise ValueError("expected contiguous q [B,H,1,D] of the cache's D")
    if prefix_table.dtype is not torch.int32:
        raise TypeError("prefix_table must be int32")
    if prefix_table.get_device() != device or prefix_table.dim() != 1 \
            or not prefix_table.is_contiguous() \
            or prefix_table.shape[0] * page_size < prefix_len:
        raise ValueError("prefix_table must name the pages of prefix_len keys, on q's device")
    H = q.shape[1]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = _output(out, q, (B, H, 1, D), q.dtype, stream, "out")
    lse = _output(lse, q, (B, H, 1), torch.float32, stream, "lse")
    ws, ws_bytes, _keep = _captured_workspace(lib, "decode_shared", q, stream, B, H, Hkv, D)
    status = lib.fn("decode_shared", _suffix(q))(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr(),
        prefix_table.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), B, H, Hkv,
        int(prefix_len), page_size, block_table.shape[1], D, scale, ws, ws_bytes,
        _stream_ptr(stream))
    _raise(lib, status)
    return out, lse


_Q8_CODES = _Q8_FLOATS = None


def _check_q8(tensors, k_cache, v_cache, k_exp, v_exp, block_table, seq_lens, starts=None):
    """What the calls on an 8-bit paged cache have in common (as in _check_paged, with codes [P, page,
    Hkv, D] of one type and exponents [P, Hkv, page] uint8): what is right is passed in one look at each
    tensor. -> code, device, B, pages, page size, Hkv, D."""
    global _Q8_CODES, _Q8_FLOATS
    torch = _torch()
    if _Q8_CODES is None:
        _Q8_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
        _Q8_FLOATS = {torch.float32, torch.float16, torch.bfloat16}
    device = torch.cuda.current_device()
    kind, uint8, int32 = k_cache.dtype, torch.uint8, torch.int32
    code = _Q8_CODES.get(kind)
    ints = (block_table, seq_lens) if starts is None else (block_table, seq_lens, starts)
    floating = tensors[0].dtype if tensors else torch.float32
    good = (code is not None and v_cache.dtype is kind and k_exp.dtype is uint8
            and v_exp.dtype is uint8 and floating in _Q8_FLOATS)
    for t in (k_cache, v_cache, k_exp, v_exp):
        if t.get_device() != device or not t.is_contiguous() or t.data_ptr() & 15:
            good = False
    for t in ints:
        if t.get_device() != device or t.dtype is not int32 or not t.is_contiguous():
            good = False
    for t in tensors:
        if t.get_device() != device or t.dtype is not floating or t.data_ptr() & 15:
            good = False
    if not good:
        _refuse_q8(tensors, (k_cache, v_cache, k_exp, v_exp), ints, device)
    shape, B = k_cache.shape, block_table.shape[0]
    if len(shape) != 4 or v_cache.shape != shape \
            or k_exp.shape != (shape[0], shape[2], shape[1]) or v_exp.shape != k_exp.shape:
        raise ValueError("expected k_cache, v_cache [P,page,Hkv,D] and k_exp, v_exp [P,Hkv,page]")
    if block_table.dim() != 2 or seq_lens.shape != (B,):
        raise ValueError("expected block_table [B,max_pages] and seq_lens [B]")
    if starts is not None and starts.shape != (B + 1,):
        raise ValueError("expected starts [B+1]")
    return (code, device, B, *shape)


def _refuse_q8(tensors, cache, ints, device):
    torch = _torch()
    if cache[0].dtype not in _Q8_CODES or cache[1].dtype != cache[0].dtype \
            or any(t.dtype != torch.uint8 for t in cache[2:]):
        raise TypeError("the caches must both be int8 or float8_e4m3fn, their exponents uint8")
    if any(t.get_device() != device for t in (*tensors, *cache, *ints)):
        raise ValueError("tensors must be on the GPU, on the current device")
    if tensors:
        _suffix(tensors[0])
    if any(t.dtype != tensors[0].dtype for t in tensors):
        raise ValueError("all tensors must share one dtype")
    if any(t.dtype != torch.int32 for t in ints):
        raise TypeError("block_table, seq_lens and query_starts must be int32")
    if not all(t.is_contiguous() for t in (*cache, *ints)):
        raise ValueError("the caches, exponents and int32 tensors must be contiguous")
    raise ValueError("tensors must start at a multiple of 16 bytes")


def _output_like(given, q, stream):
    """_output of the shape and type of q, which is contiguous: 0.5 us less where it is a new one."""
    if given is not None or stream is not None:
        return _output(given, q, q.shape, q.dtype, stream, "out")
    return _torch().empty_like(q)


def _attend_q8(lib, kind, q, stream, sizes, call):
    """call(workspace, bytes). Only a captured call is refused without a workspace, and has done nothing
    then: it gets one from the graph's pool (asking first costs every call 0.5 us of 13)."""
    status = call(None, 0)
    if status == OUT_OF_MEMORY:
        ws, ws_bytes, _keep = _captured_workspace(lib, kind, q, stream, *sizes)
        if ws is not None:
            status = call(ws, ws_bytes)
    _raise(lib, status)


def flash_attention_append_paged_q8(k, v, k_cache, v_cache, k_exp, v_exp, block_table, seq_lens,
                                    query_starts=None, q=None, cos=None, sin=None,
                                    interleaved: bool = False, out=None, stream=None,
                                    lib: Optional[CuFlashLibrary] = None):
    """flash_attention_append_paged into a cache of one byte an element: k_cache, v_cache [P, page,
    Hkv, D] int8 or float8_e4m3fn, k_exp, v_exp [P, Hkv, page] uint8; an element is its code times
    2^(exponent - 127). A head's row of a token gets the least exponent that its largest element allows
    and codes rounded to the nearest. -> rotated q [T, H, D] or None
    (cuflash_attention_append_paged_q8_*)."""
    lib = lib or load_library()
    given = (k, v) if q is None else (k, v, q)
    code, device, B, pages, page_size, Hkv, D = _check_q8(given, k_cache, v_cache, k_exp, v_exp,
                                                          block_table, seq_lens, query_starts)
    T, H = k.shape[0], 0 if q is None else q.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != (T, Hkv, D) \
            or (q is not None and q.shape != (T, H, D)):
        raise ValueError("expected k, v [T,Hkv,D] and q [T,H,D] of the cache's Hkv and D")
    positions, R = _rotation(cos, sin, device)
    k_stride, v_stride, q_stride = _token_stride(k, "k"), _token_stride(v, "v"), 0
    if q is not None:
        q_stride = _token_stride(q, "q")
        out = _output(out, q, (T, H, D), q.dtype, stream, "out")
    elif out is not None:
        raise ValueError("out is the rotated q: it needs q")
    q_ptr, out_ptr = (None, None) if q is None else (q.data_ptr(), out.data_ptr())
    cos_ptr, sin_ptr = (None, None) if cos is None else (cos.data_ptr(), sin.data_ptr())
    status = lib.fn("append_paged_q8", _suffix(k))(
        q_ptr, k.data_ptr(), v.data_ptr(), out_ptr, k_cache.data_ptr(), v_cache.data_ptr(),
        k_exp.data_ptr(), v_exp.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
        None if query_starts is None else query_starts.data_ptr(), cos_ptr, sin_ptr, T, B, H, Hkv,
        q_stride, k_stride, v_stride, pages, page_size, block_table.shape[1], D, R, positions,
        bool(interleaved), code, _stream_ptr(stream))
    _raise(lib, status)
    return out


def flash_attention_read_paged_q8(k_cache, v_cache, k_exp, v_exp, block_table, seq_lens, key_starts,
                                  num_tokens: int, dtype=None, k_out=None, v_out=None, stream=None,
                                  lib: Optional[CuFlashLibrary] = None):
    """The keys and values that an 8-bit paged cache holds, as numbers of `dtype` (bfloat16 if not
    given): tokens key_starts[b] .. key_starts[b + 1] - 1 are the newest of sequence b, as in
    flash_attention_append_paged_q8, of whose tokens it gives back what the cache has. num_tokens:
    rows of the outputs, those from key_starts[B] on are left as they are. -> k, v [num_tokens, Hkv, D]
    (cuflash_attention_read_paged_q8_*)."""
    torch = _torch()
    lib = lib or load_library()
    code, _, B, pages, page_size, Hkv, D = _check_q8((), k_cache, v_cache, k_exp, v_exp,
                                                     block_table, seq_lens, key_starts)
    if key_starts is None:
        raise ValueError("expected key_starts [B+1]")
    dtype = dtype or (torch.bfloat16 if k_out is None else k_out.dtype)
    T = int(num_tokens)
    if T < 1:
        raise CuFlashError(INVALID_DIMENSION, lib.error_string(INVALID_DIMENSION))
    k_out = _output(k_out, k_exp, (T, Hkv, D), dtype, stream, "k_out")
    v_out = _output(v_out, k_exp, (T, Hkv, D), dtype, stream, "v_out")
    status = lib.fn("read_paged_q8", _suffix(k_out))(
        k_cache.data_ptr(), v_cache.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(),
        k_out.data_ptr(), v_out.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
        key_starts.data_ptr(), T, B, Hkv, pages, page_size, block_table.shape[1], D, code,
        _stream_ptr(stream))
    _raise(lib, status)
    return k_out, v_out


def flash_attention_decode_paged_q8(q, k_cache, v_cache, k_exp, v_exp, block_table, seq_lens,
                                    scale: Optional[float] = None, out=None, lse=None, stream=None,
                                    lib: Optional[CuFlashLibrary] = None):
    """flash_attention_decode_paged over a cache of one byte an element (see
    flash_attention_append_paged_q8): q [B, H, 1, D] -> O [B, H, 1, D], L float32 [B, H, 1]
    (cuflash_attention_decode_paged_q8_*)."""
    torch = _torch()
    lib = lib or load_library()
    code, _, B, _, page_size, Hkv, D = _check_q8((q,), k_cache, v_cache, k_exp, v_exp, block_table,
                                                 seq_lens)
    if q.dim() != 4 or q.shape[0] != B or q.shape[2] != 1 or q.shape[3] != D \
            or not q.is_contiguous():
        raise ValueError("expected contiguous q [B,H,1,D] of the cache's D")
    H = q.shape[1]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = _output_like(out, q, stream)
    lse = _output(lse, q, (B, H, 1), torch.float32, stream, "lse")
    fn = lib.fn("decode_paged_q8", _suffix(q))
    _attend_q8(lib, "decode_paged_q8", q, stream, (B, H, Hkv, D), lambda ws, ws_bytes: fn(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(),
        out.data_ptr(), lse.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), B, H, Hkv,
        page_size, block_table.shape[1], D, scale, code, ws, ws_bytes, _stream_ptr(stream)))
    return out, lse


def flash_attention_forward_paged_q8(q, k_cache, v_cache, k_exp, v_exp, block_table, seq_lens,
                                     query_starts, scale: Optional[float] = None,
                                     causal: bool = False, out=None, lse=None, stream=None,
                                     lib: Optional[CuFlashLibrary] = None):
    """flash_attention_forward_paged over a cache of one byte an element (see
    flash_attention_append_paged_q8): q [T, H, D] -> O [T, H, D], L float32 [T, H]
    (cuflash_attention_forward_paged_q8_*)."""
    torch = _torch()
    lib = lib or load_library()
    code, _, B, _, page_size, Hkv, D = _check_q8((q,), k_cache, v_cache, k_exp, v_exp, block_table,
                                                 seq_lens, query_starts)
    if query_starts is None or q.dim() != 3 or q.shape[2] != D or not q.is_contiguous():
        raise ValueError("expected contiguous q [T,H,D] of the cache's D and query_starts [B+1]")
    T, H = q.shape[:2]
    scale = float(D ** -0.5) if scale is None else float(scale)
    out = _output_like(out, q, stream)
    lse = _output(lse, q, (T, H), torch.float32, stream, "lse")
    fn = lib.fn("forward_paged_q8", _suffix(q))
    _attend_q8(lib, "forward_paged_q8", q, stream, (T, B, H, Hkv, D), lambda ws, ws_bytes: fn(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(),
        out.data_ptr(), lse.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
        query_starts.data_ptr(), T, B, H, Hkv, page_size, block_table.shape[1], D, scale,
        bool(causal), code, ws, ws_bytes, _stream_ptr(stream)))
    return out, lse


__all__ = [
    "CuFlashError", "CuFlashLibrary", "EXPORTED_SYMBOLS", "load_library",
    "candidate_library_paths", "flash_attention_forward", "flash_attention_backward",
    "flash_attention_forward_ext", "flash_attention_backward_ext", "flash_attention_decode",
    "flash_attention_decode_paged", "flash_attention_append_paged",
    "flash_attention_forward_paged", "flash_attention_decode_shared", "PAGED_CACHE_SYMBOLS",
    "flash_attention_append_paged_q8", "flash_attention_read_paged_q8",
    "flash_attention_decode_paged_q8", "flash_attention_forward_paged_q8",
    "PAGED_CACHE_Q8_SYMBOLS",
    "SUCCESS", "INVALID_DIMENSION", "DIMENSION_MISMATCH",
    "NULL_POINTER", "CUDA_ERROR", "OUT_OF_MEMORY", "UNSUPPORTED_HEAD_DIM", "UNSUPPORTED_DTYPE",
]

if sys.version_info < (3, 8):  # pragma: no cover
    raise RuntimeError("python >= 3.8 required")
