"""Operator surface of the GPU KV partition over the gfx950 C-ABI library.

Thin ctypes layer: validates shapes/dtypes/devices, passes data pointers and
the current HIP stream to scope_amd/lib/libwsgpu.so (include/wsgpu.h) and
raises on any error.  There is no fallback: if the library is missing or a
tensor is not on a GPU, the call fails.

Tensor conventions (all CUDA/HIP tensors, contiguous):
  GQA pools   k_pages, v_pages  [num_pages, Hkv, page_size, D] bfloat16
  MLA pool    latent_pages      [num_pages, page_size, 576]    bfloat16
  page_table  [B, max_pages] int32, gpu_len [B] int32
  partials    (out fp32 normalised, lse fp32 natural log); empty = (0, -inf)
  8-bit pools k_pages, v_pages  [num_pages, Hkv, page_size, D] float8_e4m3fn with
              k_scale, v_scale  [num_pages, Hkv, page_size]    float8_e8m0fnu
              (one power of two per token and KV head)
"""
from __future__ import annotations

import ctypes
import functools
import os
from typing import NamedTuple

import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libwsgpu.so")

# Entry points declared in include/wsgpu.h.
EXPORTS = (
    "ws_last_error",
    "ws_version",
    "ws_kv_append",
    "ws_latent_append",
    "ws_dense_paging",
    "ws_decode_plan",
    "ws_attn_decode_plan",
    "ws_gqa_decode_partial",
    "ws_gqa_append_decode_partial",
    "ws_mla_decode_partial",
    "ws_mla_append_decode_partial",
    "ws_gqa_append_decode_split",
    "ws_gqa_decode_full",
    "ws_gqa_append_decode_full",
    "ws_mla_append_decode_split",
    "ws_merge_split",
    "ws_mla_merge_split_uv",
    "ws_split_reduce",
    "ws_lse_merge",
    "ws_attn_decode_partial",
    "ws_attn_append_decode_partial",
    "ws_copy",
    "ws_copy_pages",
    "ws_noalloc_scratch_bytes",
    "ws_gqa_append_decode_partial_noalloc",
    "ws_pages_extend",
    "ws_pages_release",
    "ws_rope",
    "ws_rope_append",
    "ws_gqa8_decode_plan",
    "ws_gqa8_decode_partial",
    "ws_gqa8_decode_full",
    "ws_gqa_prompt_plan",
    "ws_gqa_prompt",
)

# Formats of the second operand of lse_merge (include/wsgpu.h).
PARTIAL_LSE_F32 = 0
TRIPLE_UNNORM_F32 = 1
TRIPLE_NORM_BF16 = 2
TRIPLE_NORM_F32 = 3
PARTIAL_LSE_BF16 = 4

MLA_LATENT = 576
MLA_C = 512
MLA_PE = 64


class WsError(RuntimeError):
    """A libwsgpu entry point returned an error."""


_lib = None


def lib() -> ctypes.CDLL:
    """Load libwsgpu.so (torch is imported first so that the process keeps a
    single HIP runtime)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is not built; run `python -m scope_amd._build` "
                "(or __graft_entry__.build())")
        L = ctypes.CDLL(LIB_PATH)
        vp, i32, i64, f32, sz = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int64,
                                 ctypes.c_float, ctypes.c_size_t)
        L.ws_last_error.restype = ctypes.c_char_p
        L.ws_last_error.argtypes = []
        L.ws_version.restype = ctypes.c_char_p
        L.ws_version.argtypes = []
        L.ws_kv_append.restype = i32
        L.ws_kv_append.argtypes = [vp, vp, vp, vp, vp, vp, i32, i32, i32, i32,
                                   i32, i32, i32, i32, vp]
        L.ws_latent_append.restype = i32
        L.ws_latent_append.argtypes = [vp, i64, vp, i64, vp, vp, vp, i32, i32,
                                       i32, i32, i32, i32, vp]
        L.ws_dense_paging.restype = i32
        L.ws_dense_paging.argtypes = [vp, vp, i32, i32, vp, i64, vp]
        L.ws_decode_plan.restype = i32
        L.ws_decode_plan.argtypes = [i32, i32, i32, i32, i32,
                                     ctypes.POINTER(i32), ctypes.POINTER(sz)]
        L.ws_attn_decode_plan.restype = i32
        L.ws_attn_decode_plan.argtypes = [i32, i32, i32, i32, i32, i32,
                                          ctypes.POINTER(i32), ctypes.POINTER(sz)]
        L.ws_gqa_decode_partial.restype = i32
        L.ws_gqa_decode_partial.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32,
                                            i32, i32, i32, i32, i32, i32, f32,
                                            vp, vp, vp, sz, vp]
        L.ws_gqa_append_decode_partial.restype = i32
        L.ws_gqa_append_decode_partial.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp,
                                                   i32, i32, i32, i32, i32, i32, i32,
                                                   i32, i32, f32, vp, vp, vp, sz, vp]
        L.ws_gqa_decode_full.restype = i32
        L.ws_gqa_decode_full.argtypes = [vp] * 5 + [i32] * 9 + [f32, vp, vp, vp, vp, sz, vp]
        L.ws_gqa_append_decode_full.restype = i32
        L.ws_gqa_append_decode_full.argtypes = [vp] * 8 + [i32] * 9 + [f32, vp, vp, vp, vp, sz,
                                                                        vp]
        L.ws_mla_decode_partial.restype = i32
        L.ws_mla_decode_partial.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32,
                                            i32, i32, i32, i32, f32, vp, vp,
                                            vp, sz, vp]
        L.ws_mla_append_decode_partial.restype = i32
        L.ws_mla_append_decode_partial.argtypes = [vp, vp, vp, i64, vp, i64, vp, vp,
                                                   vp, vp, i32, i32, i32, i32, i32,
                                                   i32, i32, f32, vp, vp, vp, sz, vp]
        L.ws_gqa_append_decode_split.restype = i32
        L.ws_gqa_append_decode_split.argtypes = L.ws_gqa_append_decode_partial.argtypes
        L.ws_mla_append_decode_split.restype = i32
        L.ws_mla_append_decode_split.argtypes = L.ws_mla_append_decode_partial.argtypes
        L.ws_merge_split.restype = i32
        L.ws_merge_split.argtypes = [vp, i32, i32, i32, i32, i32, i32, vp, vp, vp, sz,
                                     vp, vp, vp, i32, vp, vp, vp, vp]
        L.ws_mla_merge_split_uv.restype = i32
        L.ws_mla_merge_split_uv.argtypes = [vp, i32, i32, i32, i32, vp, vp, vp, sz, vp, vp, vp,
                                            i32, vp, i32, vp, vp, vp, vp]
        L.ws_split_reduce.restype = i32
        L.ws_split_reduce.argtypes = [vp, vp, vp, i32, i32, i32, i32, i32, vp,
                                      vp, vp]
        L.ws_attn_decode_partial.restype = i32
        L.ws_attn_decode_partial.argtypes = [vp] * 5 + [i32] * 10 + [f32, vp, vp, vp, sz, vp]
        L.ws_attn_append_decode_partial.restype = i32
        L.ws_attn_append_decode_partial.argtypes = [vp] * 8 + [i32] * 10 + [f32, vp, vp, vp,
                                                                             sz, vp]
        L.ws_copy.restype = i32
        L.ws_copy.argtypes = [vp, vp, sz, vp]
        L.ws_copy_pages.restype = i32
        L.ws_copy_pages.argtypes = [vp, i64, vp, i32, vp, i64, vp, i32, i32, i32, i64, i32, vp]
        L.ws_noalloc_scratch_bytes.restype = sz
        L.ws_noalloc_scratch_bytes.argtypes = []
        L.ws_gqa_append_decode_partial_noalloc.restype = i32
        L.ws_gqa_append_decode_partial_noalloc.argtypes = [vp] * 8 + [i32] * 9 + [f32, vp, vp,
                                                                               vp]
        L.ws_lse_merge.restype = i32
        L.ws_lse_merge.argtypes = [vp, vp, vp, vp, vp, i32, vp, vp, vp, i32,
                                   i32, vp]
        L.ws_pages_extend.restype = i32
        L.ws_pages_extend.argtypes = [vp] * 11 + [i32] * 6 + [vp]
        L.ws_pages_release.restype = i32
        L.ws_pages_release.argtypes = [vp] * 7 + [i32] * 4 + [vp]
        L.ws_rope.restype = i32
        L.ws_rope.argtypes = [vp, i64, vp, i64, vp, i32, vp, ctypes.c_char_p, i32, f32, vp, vp] + \
            [i32] * 5 + [vp]
        L.ws_rope_append.restype = i32
        L.ws_rope_append.argtypes = [vp, i64, vp, i64, vp, i64, vp, i32, vp, ctypes.c_char_p, i32,
                                     f32, vp, vp, vp, vp, vp, vp] + [i32] * 7 + [vp]
        L.ws_gqa8_decode_plan.restype = i32
        L.ws_gqa8_decode_plan.argtypes = [i32] * 5 + [ctypes.POINTER(i32), ctypes.POINTER(sz)]
        L.ws_gqa8_decode_partial.restype = i32
        L.ws_gqa8_decode_partial.argtypes = [vp] * 7 + [i32] * 9 + [f32, vp, vp, vp, sz, vp]
        L.ws_gqa8_decode_full.restype = i32
        L.ws_gqa8_decode_full.argtypes = [vp] * 7 + [i32] * 9 + [f32, vp, vp, vp, vp, sz, vp]
        L.ws_gqa_prompt_plan.restype = i32
        L.ws_gqa_prompt_plan.argtypes = [i32] * 8 + [ctypes.POINTER(i32), ctypes.POINTER(sz)]
        L.ws_gqa_prompt.restype = i32
        L.ws_gqa_prompt.argtypes = [vp] * 8 + [i32] * 10 + [f32, vp, vp, vp, vp, sz, vp]
        _lib = L
    return _lib


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise WsError(f"{name}: {lib().ws_last_error().decode()} (rc={rc})")


# Addresses go to the library as plain integers: the argtypes convert them, and
# a c_void_p object per argument cost 0.2 us each.
def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device: torch.device):
    """The current HIP stream of `device` (the raw handle torch launches on)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(idx)


def _require(t: torch.Tensor, name: str, dtype: torch.dtype, device=None,
             ndim=None, contiguous=True) -> None:
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda
            and (device is None or t.device == device) and (ndim is None or t.dim() == ndim)
            and (not contiguous or t.is_contiguous())):
        return
    # what is wrong, in this order
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (got {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims (got {tuple(t.shape)})")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# ---------------------------------------------------------------------------
# workspace

_workspaces: dict = {}


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch for the split partials of the one-launch entry points, one per
    (device, stream): calls on one stream reuse it in stream order, calls on
    different streams never share it.  Grown on demand (the old buffer is
    freed through torch's stream-ordered allocator, so a launch still
    queued on this stream keeps its memory until it ran).  Each call writes
    the slots it reads back, so no initial contents are needed."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    key = (idx, torch._C._cuda_getCurrentRawStream(idx))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


_plans: dict = {}


def dense_paging(n: int, tokens: int, ones_shape, device):
    """(page_table [n, 1], lengths [n], ones) of n contiguous per-row buffers
    that hold `tokens` tokens each (ws_dense_paging)."""
    ints = torch.empty((2, n), dtype=torch.int32, device=device)
    ones = torch.empty(ones_shape, dtype=torch.float32, device=device)
    if not ints.is_cuda:
        raise ValueError(f"device must be a GPU (got {device})")
    _check(lib().ws_dense_paging(ints.data_ptr(), ints.data_ptr() + 4 * n, n, tokens,
                                 _ptr(ones), ones.numel(), _stream(ints.device)),
           "ws_dense_paging")
    return ints[0].view(n, 1), ints[1], ones


def decode_plan(kind: int, rows_kv: int, heads: int, max_len: int,
                n_workgroups: int = 0):
    """(n_splits, workspace_bytes) of a decode call: kind 0 = GQA
    (rows_kv = B * Hkv, heads = group size), 1 = MLA (rows_kv = B, heads = 16).
    A split is one wave for GQA and one workgroup for MLA; the keyword keeps
    the name n_workgroups.  0 lets the library choose for the current
    device."""
    # the answer depends on the arguments and the current device only (a
    # decode loop asks the same question for every layer of a step)
    key = (kind, rows_kv, heads, max_len, n_workgroups,
           torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -1)
    hit = _plans.get(key)
    if hit is not None:
        return hit
    n, wsb = ctypes.c_int(0), ctypes.c_size_t(0)
    _check(lib().ws_decode_plan(kind, rows_kv, heads, max_len, n_workgroups,
                                ctypes.byref(n), ctypes.byref(wsb)), "ws_decode_plan")
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = (n.value, wsb.value)
    return n.value, wsb.value


def gqa_plan(rows_kv: int, heads: int, Dk: int, Dv: int, max_len: int,
             n_workgroups: int = 0):
    """decode_plan kind 0 at key width Dk and value width Dv
    (ws_attn_decode_plan; kind 0 itself sizes the workspace for 128)."""
    if Dk == 128 and Dv == 128:
        return decode_plan(0, rows_kv, heads, max_len, n_workgroups)
    key = ("attn", rows_kv, heads, Dk, Dv, max_len, n_workgroups,
           torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -1)
    hit = _plans.get(key)
    if hit is not None:
        return hit
    n, wsb = ctypes.c_int(0), ctypes.c_size_t(0)
    _check(lib().ws_attn_decode_plan(rows_kv, heads, Dk, Dv, max_len, n_workgroups,
                                     ctypes.byref(n), ctypes.byref(wsb)),
           "ws_attn_decode_plan")
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = (n.value, wsb.value)
    return n.value, wsb.value


# ---------------------------------------------------------------------------
# transfers


def copy_(dst: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """dst.copy_(src) by the library's copy kernel (ws_copy) on the current
    stream of the GPU side: one of them on the GPU, the other on the GPU or in
    pinned host memory.  Used for a layer's query to the host partial, where
    a DMA copy's set-up latency sits on every layer's critical path."""
    if dst.dtype != src.dtype or dst.numel() != src.numel():
        raise ValueError("copy_: dst and src must have the same dtype and size")
    gpu = dst if dst.is_cuda else src
    if not gpu.is_cuda:
        raise ValueError("copy_: one side must be on a GPU")
    for t, n in ((dst, "dst"), (src, "src")):
        if not t.is_contiguous():
            raise ValueError(f"copy_: {n} must be contiguous")
        if t.is_cuda and t.device != gpu.device:
            raise ValueError("copy_: tensors on two GPUs")
        if not t.is_cuda and not t.is_pinned():
            raise ValueError(f"copy_: {n} must be on the GPU or in pinned host memory")
    _check(lib().ws_copy(_ptr(dst), _ptr(src), dst.numel() * dst.element_size(),
                         _stream(gpu.device)), "ws_copy")
    return dst


def copy_pages(dst_pool: torch.Tensor, dst_ids, src_pool: torch.Tensor, src_ids,
               max_workgroups: int = 0) -> None:
    """dst_pool[:, dst_ids[i]] = src_pool[:, src_ids[i]] for every layer, by
    the library's page-copy kernel (ws_copy_pages) on the current stream of
    the GPU side.  Pools are [layers, num_pages, *page] of one dtype; one of
    them on the GPU, the other on the same GPU or in pinned host memory (the
    kernel crosses the host link itself: no host gather, no staging).
    max_workgroups bounds the kernel's grid (0: the library's default)."""
    if dst_pool.dtype != src_pool.dtype or dst_pool.dim() < 2 or \
            dst_pool.shape[0] != src_pool.shape[0] or dst_pool.shape[2:] != src_pool.shape[2:]:
        raise ValueError("copy_pages: pools must match in dtype, layers and page shape")
    gpu = dst_pool if dst_pool.is_cuda else src_pool
    if not gpu.is_cuda:
        raise ValueError("copy_pages: one pool must be on a GPU")
    for t, n in ((dst_pool, "dst_pool"), (src_pool, "src_pool")):
        if not t.is_contiguous():
            raise ValueError(f"copy_pages: {n} must be contiguous")
        if t.is_cuda and t.device != gpu.device:
            raise ValueError("copy_pages: pools on two GPUs")
        if not t.is_cuda and not t.is_pinned():
            raise ValueError(f"copy_pages: {n} must be on the GPU or in pinned host memory")
    di = np.asarray(dst_ids, np.int64).reshape(-1)
    si = np.asarray(src_ids, np.int64).reshape(-1)
    if di.shape != si.shape:
        raise ValueError("copy_pages: dst_ids and src_ids differ in length")
    if di.size == 0:
        return
    for ids, pool, n in ((di, dst_pool, "dst_ids"), (si, src_pool, "src_ids")):
        if ids.min() < 0 or ids.max() >= pool.shape[1]:
            raise ValueError(f"copy_pages: {n} outside [0, {pool.shape[1]})")
    ids = torch.from_numpy(np.stack([di, si]).astype(np.int32)).to(gpu.device)
    page_bytes = dst_pool[0, 0].numel() * dst_pool.element_size()
    _check(lib().ws_copy_pages(
        _ptr(dst_pool), dst_pool.stride(0) * dst_pool.element_size(), _ptr(ids[0]),
        dst_pool.shape[1], _ptr(src_pool), src_pool.stride(0) * src_pool.element_size(),
        _ptr(ids[1]), src_pool.shape[1], int(di.size), dst_pool.shape[0], page_bytes,
        int(max_workgroups), _stream(gpu.device)), "ws_copy_pages")


# ---------------------------------------------------------------------------
# append


def kv_append(k_new, v_new, k_pages, v_pages, page_table, gpu_len, update_len=True):
    """Write k_new/v_new [B, Hkv, n_new, D] at slots gpu_len[b].. of each
    sequence's pages (bit copies), then gpu_len += n_new if update_len."""
    dev = k_pages.device
    _require(k_new, "k_new", torch.bfloat16, dev, 4)
    _require(v_new, "v_new", torch.bfloat16, dev, 4)
    _require(k_pages, "k_pages", torch.bfloat16, dev, 4)
    _require(v_pages, "v_pages", torch.bfloat16, dev, 4)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    B, Hkv, n_new, D = k_new.shape
    P, Hkv2, PS, D2 = k_pages.shape
    if v_new.shape != k_new.shape or v_pages.shape != k_pages.shape:
        raise ValueError("k/v shapes differ")
    if Hkv2 != Hkv or D2 != D or page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError(
            f"shape mismatch: new {tuple(k_new.shape)} pages {tuple(k_pages.shape)} "
            f"page_table {tuple(page_table.shape)} gpu_len {tuple(gpu_len.shape)}")
    _check(lib().ws_kv_append(_ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages),
                              _ptr(page_table), _ptr(gpu_len), B, Hkv, D, n_new, PS,
                              page_table.shape[1], P, int(bool(update_len)),
                              _stream(dev)), "ws_kv_append")


def latent_append(c_new, pe_new, latent_pages, page_table, gpu_len, update_len=True):
    """Write c_new [B, n_new, 512] and pe_new [B, n_new, 64] as the 576-wide
    latent at slots gpu_len[b].. of each sequence's pages."""
    dev = latent_pages.device
    for t, n in ((c_new, "c_new"), (pe_new, "pe_new")):
        _require(t, n, torch.bfloat16, dev, 3, contiguous=False)
        if t.stride(2) != 1 or t.stride(0) != t.shape[1] * t.stride(1):
            raise ValueError(f"{n} must be [B, n, W] with unit last stride and "
                             "batch stride n * row stride")
    _require(latent_pages, "latent_pages", torch.bfloat16, dev, 3)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    B, n_new, W = c_new.shape
    P, PS, L = latent_pages.shape
    if W != MLA_C or pe_new.shape != (B, n_new, MLA_PE) or L != MLA_LATENT:
        raise ValueError("latent layout is 512 c_kv + 64 k_pe = 576")
    if page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError("page_table/gpu_len batch mismatch")
    _check(lib().ws_latent_append(_ptr(c_new), c_new.stride(1), _ptr(pe_new),
                                  pe_new.stride(1), _ptr(latent_pages), _ptr(page_table),
                                  _ptr(gpu_len), B, n_new, PS, page_table.shape[1], P,
                                  int(bool(update_len)), _stream(dev)),
           "ws_latent_append")


# ---------------------------------------------------------------------------
# decode partials


def gqa_decode_partial(q, k_pages, v_pages, page_table, gpu_len, scale, max_len,
                       n_workgroups=0, out=None, lse=None):
    """Split-KV GQA decode attention over the pooled tokens.

    q [B, Hq, D] bf16 -> (out [B, Hq, D] fp32 normalised, lse [B, Hq] fp32).
    max_len must bound every gpu_len[b] (the host's mirror of the lengths).
    """
    dev = k_pages.device
    _require(q, "q", torch.bfloat16, dev, 3)
    _require(k_pages, "k_pages", torch.bfloat16, dev, 4)
    _require(v_pages, "v_pages", torch.bfloat16, dev, 4)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D:
        raise ValueError("k/v page pools must match q's head_dim")
    if page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError("page_table/gpu_len batch mismatch")
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    _require(out, "out", torch.float32, dev, 3)
    _require(lse, "lse", torch.float32, dev, 2)
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, D, D, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    _run("ws_gqa_decode_partial", dev, _ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
         _ptr(gpu_len), B, Hq, Hkv, D, PS, page_table.shape[1], P, int(max_len), nwg, float(scale),
         _ptr(out), _ptr(lse), _ptr(ws), wsb)
    return out, lse


def gqa_decode_full(q, k_pages, v_pages, page_table, gpu_len, scale, max_len,
                    n_workgroups=0, out_bf16=None, lse=None):
    """gqa_decode_partial for a partition that holds every token: returns
    (out [B, Hq, D] bf16, the rounded fp32 output; lse [B, Hq] fp32)."""
    dev = _gpu(k_pages, "k_pages")
    _require_all(dev, _DECODE16_ARGS, (q, k_pages, v_pages, page_table, gpu_len))
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match the pools {tuple(k_pages.shape)}")
    if page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError("page_table/gpu_len batch mismatch")
    if out_bf16 is None:
        out_bf16 = torch.empty_like(q)
    else:
        _require(out_bf16, "out_bf16", torch.bfloat16, dev, 3)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    else:
        _require(lse, "lse", torch.float32, dev, 2)
    if out_bf16.shape != q.shape or lse.shape != (B, Hq):
        raise ValueError("out_bf16 must be [B, Hq, D] and lse [B, Hq]")
    if B == 0:
        return out_bf16, lse
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, D, D, int(max_len), int(n_workgroups))
    wsb = (wsb + 255) & ~255
    # the call's own, with the fp32 output behind the pieces
    ws = torch.empty(wsb + 4 * B * Hq * D, dtype=torch.uint8, device=dev)
    _run("ws_gqa_decode_full", dev, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
         page_table.data_ptr(), gpu_len.data_ptr(), B, Hq, Hkv, D, PS, page_table.shape[1], P,
         int(max_len), nwg, float(scale), out_bf16.data_ptr(), ws.data_ptr() + wsb, lse.data_ptr(),
         ws.data_ptr(), wsb)
    return out_bf16, lse


def attn_decode_partial(q, k_pages, v_pages, page_table, gpu_len, scale, max_len,
                        n_workgroups=0, k_new=None, v_new=None, len_out=None, out=None,
                        lse=None):
    """Decode attention with separate key / value widths (ws_attn_decode_partial,
    or ws_attn_append_decode_partial with k_new / v_new): q [B, Hq, Dk],
    k_pages [P, Hkv, PS, Dk], v_pages [P, Hkv, PS, Dv] bf16 ->
    (out [B, Hq, Dv] fp32 normalised, lse [B, Hq] fp32).  (Dk, Dv) is
    (64, 64), (128, 128), (256, 256), or (192, 128) with one query head
    per KV head.  With k_new [B, Hkv, 1, Dk] / v_new [B, Hkv, 1, Dv], token
    gpu_len[b] is appended
    first (fused step; len_out gets the new lengths, max_len must bound
    gpu_len + 1)."""
    dev = k_pages.device
    _require(q, "q", torch.bfloat16, dev, 3)
    _require(k_pages, "k_pages", torch.bfloat16, dev, 4)
    _require(v_pages, "v_pages", torch.bfloat16, dev, 4)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    B, Hq, Dk = q.shape
    P, Hkv, PS, Dk2 = k_pages.shape
    Dv = v_pages.shape[3]
    if Dk2 != Dk or v_pages.shape[:3] != k_pages.shape[:3]:
        raise ValueError(f"pools {tuple(k_pages.shape)} / {tuple(v_pages.shape)} do not "
                         f"match q {tuple(q.shape)}")
    if page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError("page_table/gpu_len batch mismatch")
    if out is None:
        out = torch.empty((B, Hq, Dv), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    _require(out, "out", torch.float32, dev, 3)
    _require(lse, "lse", torch.float32, dev, 2)
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, Dk, Dv, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    tail = (B, Hq, Hkv, Dk, Dv, PS, page_table.shape[1], P, int(max_len), nwg, float(scale),
            _ptr(out), _ptr(lse), _ptr(ws), wsb, _stream(dev))
    if k_new is None:
        _check(lib().ws_attn_decode_partial(_ptr(q), _ptr(k_pages), _ptr(v_pages),
                                            _ptr(page_table), _ptr(gpu_len), *tail),
               "ws_attn_decode_partial")
        return out, lse
    _require(k_new, "k_new", torch.bfloat16, dev, 4)
    _require(v_new, "v_new", torch.bfloat16, dev, 4)
    if k_new.shape != (B, Hkv, 1, Dk) or v_new.shape != (B, Hkv, 1, Dv):
        raise ValueError(f"k_new / v_new must be [B, Hkv, 1, Dk] / [B, Hkv, 1, Dv]")
    if len_out is not None:
        _require(len_out, "len_out", torch.int32, dev, 1)
        if len_out.shape[0] != B or len_out.data_ptr() == gpu_len.data_ptr():
            raise ValueError("len_out must be a separate [B] int32 tensor")
    _check(lib().ws_attn_append_decode_partial(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
        _ptr(gpu_len), _ptr(len_out), *tail), "ws_attn_append_decode_partial")
    return out, lse


def mla_decode_partial(q_nope, q_pe, latent_pages, page_table, gpu_len, scale, max_len,
                       n_workgroups=0, out=None, lse=None):
    """Split-KV absorbed-MLA decode attention over the pooled latents.

    q_nope [B*H, 512] bf16 (W_UK-absorbed), q_pe [B*H, 64] bf16 ->
    (out [B*H, 512] fp32 normalised, lse [B*H] fp32).
    """
    dev = latent_pages.device
    _require(q_nope, "q_nope", torch.bfloat16, dev, 2)
    _require(q_pe, "q_pe", torch.bfloat16, dev, 2)
    _require(latent_pages, "latent_pages", torch.bfloat16, dev, 3)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    P, PS, L = latent_pages.shape
    B = page_table.shape[0]
    rows = q_nope.shape[0]
    if L != MLA_LATENT or q_nope.shape[1] != MLA_C or q_pe.shape != (rows, MLA_PE):
        raise ValueError("MLA layout is q_nope 512 + q_pe 64 over a 576 latent")
    if B == 0 or rows % B or gpu_len.shape[0] != B:
        raise ValueError("rows must be B * H with B = page_table.shape[0]")
    H = rows // B
    if out is None:
        out = torch.empty((rows, MLA_C), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((rows,), dtype=torch.float32, device=dev)
    _require(out, "out", torch.float32, dev, 2)
    _require(lse, "lse", torch.float32, dev, 1)
    nwg, wsb = decode_plan(1, B, H, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    _check(lib().ws_mla_decode_partial(
        _ptr(q_nope), _ptr(q_pe), _ptr(latent_pages), _ptr(page_table), _ptr(gpu_len),
        B, H, PS, page_table.shape[1], P, int(max_len), nwg, float(scale),
        _ptr(out), _ptr(lse), _ptr(ws), wsb, _stream(dev)), "ws_mla_decode_partial")
    return out, lse


def gqa_append_decode_partial(q, k_new, v_new, k_pages, v_pages, page_table, len_in,
                              len_out, scale, max_len, n_workgroups=0, out=None,
                              lse=None):
    """Append k_new/v_new [B, Hkv, 1, D] at position len_in[b] of each sequence
    and attend over the partition including it, in one launch.  len_out[b] =
    len_in[b] + 1 (len_out may be None; it must not be len_in).  max_len must
    bound every len_in[b] + 1.  Returns (out [B, Hq, D] fp32, lse [B, Hq])."""
    dev = k_pages.device
    _require(q, "q", torch.bfloat16, dev, 3)
    _require(k_new, "k_new", torch.bfloat16, dev, 4)
    _require(v_new, "v_new", torch.bfloat16, dev, 4)
    _require(k_pages, "k_pages", torch.bfloat16, dev, 4)
    _require(v_pages, "v_pages", torch.bfloat16, dev, 4)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(len_in, "len_in", torch.int32, dev, 1)
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D:
        raise ValueError("k/v page pools must match q's head_dim")
    if k_new.shape != (B, Hkv, 1, D) or v_new.shape != k_new.shape:
        raise ValueError(f"k_new/v_new must be [B, Hkv, 1, D] = {(B, Hkv, 1, D)}")
    if page_table.shape[0] != B or len_in.shape[0] != B:
        raise ValueError("page_table/len_in batch mismatch")
    if len_out is not None:
        _require(len_out, "len_out", torch.int32, dev, 1)
        if len_out.shape[0] != B or len_out.data_ptr() == len_in.data_ptr():
            raise ValueError("len_out must be a separate [B] int32 tensor")
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    _require(out, "out", torch.float32, dev, 3)
    _require(lse, "lse", torch.float32, dev, 2)
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, D, D, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    _check(lib().ws_gqa_append_decode_partial(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
        _ptr(len_in), _ptr(len_out), B, Hq, Hkv, D, PS, page_table.shape[1], P,
        int(max_len), nwg, float(scale), _ptr(out), _ptr(lse), _ptr(ws), wsb,
        _stream(dev)), "ws_gqa_append_decode_partial")
    return out, lse


def gqa_append_decode_full(q, k_new, v_new, k_pages, v_pages, page_table, len_in, len_out,
                           scale, max_len, n_workgroups=0, out_bf16=None, out=None, lse=None,
                           want_fp32=False):
    """The whole decode step of a partition that holds every token (no host
    share): gqa_append_decode_partial that also writes the normalised output
    in bf16 (the step launch and its combine launch).  Returns (out_bf16
    [B, Hq, D], lse [B, Hq]) or, with want_fp32 (or an `out` given),
    (out_bf16, out fp32, lse)."""
    dev = k_pages.device
    for t, n, dt, nd in ((q, "q", torch.bfloat16, 3), (k_new, "k_new", torch.bfloat16, 4),
                         (v_new, "v_new", torch.bfloat16, 4),
                         (k_pages, "k_pages", torch.bfloat16, 4),
                         (v_pages, "v_pages", torch.bfloat16, 4),
                         (page_table, "page_table", torch.int32, 2),
                         (len_in, "len_in", torch.int32, 1)):
        _require(t, n, dt, dev, nd)
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D:
        raise ValueError("k/v page pools must match q's head_dim")
    if k_new.shape != (B, Hkv, 1, D) or v_new.shape != k_new.shape:
        raise ValueError(f"k_new/v_new must be [B, Hkv, 1, D] = {(B, Hkv, 1, D)}")
    if page_table.shape[0] != B or len_in.shape[0] != B:
        raise ValueError("page_table/len_in batch mismatch")
    if len_out is not None:
        _require(len_out, "len_out", torch.int32, dev, 1)
        if len_out.shape[0] != B or len_out.data_ptr() == len_in.data_ptr():
            raise ValueError("len_out must be a separate [B] int32 tensor")
    if out_bf16 is None:
        out_bf16 = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=dev)
    _require(out_bf16, "out_bf16", torch.bfloat16, dev, 3)
    give_fp32 = want_fp32 or out is not None
    if out is None:  # the step's fp32 partial (finalised in place by the combine)
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    _require(out, "out", torch.float32, dev, 3)
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    _require(lse, "lse", torch.float32, dev, 2)
    if out_bf16.shape != q.shape or out.shape != q.shape or lse.shape != (B, Hq):
        raise ValueError("out_bf16/out must be [B, Hq, D] and lse [B, Hq]")
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, D, D, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    _check(lib().ws_gqa_append_decode_full(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
        _ptr(len_in), _ptr(len_out), B, Hq, Hkv, D, PS, page_table.shape[1], P,
        int(max_len), nwg, float(scale), _ptr(out_bf16), _ptr(out), _ptr(lse), _ptr(ws), wsb,
        _stream(dev)), "ws_gqa_append_decode_full")
    return (out_bf16, out, lse) if give_fp32 else (out_bf16, lse)


def gqa_append_decode_partial_noalloc(q, k_new, v_new, k_pages, v_pages, page_table, len_in,
                                      len_out, scale, max_len, out, lse, n_workgroups=0):
    """gqa_append_decode_partial without a workspace or any allocation: the
    caller passes out [B, Hq, D] fp32 and lse [B, Hq] fp32, and the split
    pieces live in the library's static scratch (ws_noalloc_scratch_bytes()
    per GPU).  Calls that overlap on one GPU race on that scratch; calls on
    one stream do not.  Usable under HIP graph capture."""
    dev = k_pages.device
    for t, n, dt, nd in ((q, "q", torch.bfloat16, 3), (k_new, "k_new", torch.bfloat16, 4),
                         (v_new, "v_new", torch.bfloat16, 4), (k_pages, "k_pages", torch.bfloat16, 4),
                         (v_pages, "v_pages", torch.bfloat16, 4),
                         (page_table, "page_table", torch.int32, 2),
                         (len_in, "len_in", torch.int32, 1), (out, "out", torch.float32, 3),
                         (lse, "lse", torch.float32, 2)):
        _require(t, n, dt, dev, nd)
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D or out.shape != q.shape or \
            lse.shape != (B, Hq):
        raise ValueError("k/v pools, out and lse must match q")
    if k_new.shape != (B, Hkv, 1, D) or v_new.shape != k_new.shape:
        raise ValueError(f"k_new/v_new must be [B, Hkv, 1, D] = {(B, Hkv, 1, D)}")
    if page_table.shape[0] != B or len_in.shape[0] != B:
        raise ValueError("page_table/len_in batch mismatch")
    if len_out is not None:
        _require(len_out, "len_out", torch.int32, dev, 1)
        if len_out.shape[0] != B or len_out.data_ptr() == len_in.data_ptr():
            raise ValueError("len_out must be a separate [B] int32 tensor")
    _check(lib().ws_gqa_append_decode_partial_noalloc(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
        _ptr(len_in), _ptr(len_out), B, Hq, Hkv, D, PS, page_table.shape[1], P, int(max_len),
        int(n_workgroups), float(scale), _ptr(out), _ptr(lse), _stream(dev)),
        "ws_gqa_append_decode_partial_noalloc")
    return out, lse


def mla_append_decode_partial(q_nope, q_pe, c_new, pe_new, latent_pages, page_table,
                              len_in, len_out, scale, max_len, n_workgroups=0,
                              out=None, lse=None):
    """Append the new latent (c_new [B, 1, 512], pe_new [B, 1, 64], unit last
    stride) at position len_in[b] and attend over the partition including it.
    Returns (out [B*H, 512] fp32, lse [B*H])."""
    dev = latent_pages.device
    _require(q_nope, "q_nope", torch.bfloat16, dev, 2)
    _require(q_pe, "q_pe", torch.bfloat16, dev, 2)
    _require(latent_pages, "latent_pages", torch.bfloat16, dev, 3)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(len_in, "len_in", torch.int32, dev, 1)
    B = page_table.shape[0]
    for t, n, w in ((c_new, "c_new", MLA_C), (pe_new, "pe_new", MLA_PE)):
        _require(t, n, torch.bfloat16, dev, 3, contiguous=False)
        if t.shape != (B, 1, w) or t.stride(2) != 1:
            raise ValueError(f"{n} must be [B, 1, {w}] with unit last stride")
    P, PS, L = latent_pages.shape
    rows = q_nope.shape[0]
    if L != MLA_LATENT or q_nope.shape[1] != MLA_C or q_pe.shape != (rows, MLA_PE):
        raise ValueError("MLA layout is q_nope 512 + q_pe 64 over a 576 latent")
    if B == 0 or rows % B or len_in.shape[0] != B:
        raise ValueError("rows must be B * H with B = page_table.shape[0]")
    if len_out is not None:
        _require(len_out, "len_out", torch.int32, dev, 1)
        if len_out.shape[0] != B or len_out.data_ptr() == len_in.data_ptr():
            raise ValueError("len_out must be a separate [B] int32 tensor")
    H = rows // B
    if out is None:
        out = torch.empty((rows, MLA_C), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((rows,), dtype=torch.float32, device=dev)
    nwg, wsb = decode_plan(1, B, H, int(max_len), int(n_workgroups))
    ws = _workspace(dev, wsb)
    _check(lib().ws_mla_append_decode_partial(
        _ptr(q_nope), _ptr(q_pe), _ptr(c_new), c_new.stride(0), _ptr(pe_new),
        pe_new.stride(0), _ptr(latent_pages), _ptr(page_table), _ptr(len_in),
        _ptr(len_out), B, H, PS, page_table.shape[1], P, int(max_len), nwg, float(scale),
        _ptr(out), _ptr(lse), _ptr(ws), wsb, _stream(dev)), "ws_mla_append_decode_partial")
    return out, lse


class SplitStep:
    """A deferred-combine decode step: its GPU pieces (out_g/lse_g finals and
    the split partials in `workspace`) wait for merge_split.  Holds every
    buffer the merge reads, so the step's workspace is not reused early."""

    def __init__(self, gpu_len, B, rows_per_seq, heads, Dv, cap, nwg, out_g, lse_g,
                 workspace):
        self.gpu_len, self.B, self.rows_per_seq, self.heads = gpu_len, B, rows_per_seq, heads
        self.Dv, self.cap, self.nwg = Dv, cap, nwg
        self.out_g, self.lse_g, self.workspace = out_g, lse_g, workspace
        self.guard = None  # set by an owner that reuses the workspace

    def check_workspace(self):
        if self.guard is not None and not self.guard():
            raise RuntimeError("this step's workspace was reused by a later step before "
                               "its merge")


def gqa_append_decode_split(q, k_new, v_new, k_pages, v_pages, page_table, len_in,
                            len_out, scale, max_len, n_workgroups=0, workspace=None):
    """Deferred-combine fused step (ws_gqa_append_decode_split): append and
    attend like gqa_append_decode_partial, but rows spread over several
    splits (waves) are combined later by merge_split.  len_out is required (the
    merge reads the post-step lengths).  Returns a SplitStep."""
    dev = k_pages.device
    _require(q, "q", torch.bfloat16, dev, 3)
    _require(k_new, "k_new", torch.bfloat16, dev, 4)
    _require(v_new, "v_new", torch.bfloat16, dev, 4)
    _require(k_pages, "k_pages", torch.bfloat16, dev, 4)
    _require(v_pages, "v_pages", torch.bfloat16, dev, 4)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(len_in, "len_in", torch.int32, dev, 1)
    _require(len_out, "len_out", torch.int32, dev, 1)
    B, Hq, D = q.shape
    P, Hkv, PS, D2 = k_pages.shape
    if v_pages.shape != k_pages.shape or D2 != D:
        raise ValueError("k/v page pools must match q's head_dim")
    if k_new.shape != (B, Hkv, 1, D) or v_new.shape != k_new.shape:
        raise ValueError(f"k_new/v_new must be [B, Hkv, 1, D] = {(B, Hkv, 1, D)}")
    if page_table.shape[0] != B or len_in.shape[0] != B or len_out.shape[0] != B:
        raise ValueError("page_table/len_in/len_out batch mismatch")
    if len_out.data_ptr() == len_in.data_ptr():
        raise ValueError("len_out must be a separate [B] int32 tensor")
    out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    nwg, wsb = gqa_plan(B * Hkv, Hq // Hkv, D, D, int(max_len), int(n_workgroups))
    if workspace is None:
        workspace = torch.zeros(max(wsb, 256), dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < wsb:
        raise ValueError(f"workspace needs {wsb} bytes")
    return _gqa_split_launch(q, k_new, v_new, k_pages, v_pages, page_table, len_in, len_out,
                             scale, max_len, nwg, out, lse, workspace)


def _gqa_split_launch(q, k_new, v_new, k_pages, v_pages, page_table, len_in, len_out, scale,
                      max_len, nwg, out, lse, workspace) -> SplitStep:
    """The ws_gqa_append_decode_split launch on arguments already checked
    (gqa_append_decode_split, or a cache that owns the pools, page table,
    lengths, partial buffers and workspace); returns the SplitStep."""
    B, Hq, D = q.shape
    P, Hkv, PS, _ = k_pages.shape
    _check(lib().ws_gqa_append_decode_split(
        _ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), _ptr(page_table),
        _ptr(len_in), _ptr(len_out), B, Hq, Hkv, D, PS, page_table.shape[1], P,
        int(max_len), nwg, float(scale), _ptr(out), _ptr(lse), _ptr(workspace),
        workspace.numel() * workspace.element_size(), _stream(k_pages.device)),
        "ws_gqa_append_decode_split")
    return SplitStep(len_out, B, Hkv, Hq // Hkv, D, PS * page_table.shape[1], nwg, out, lse,
                     workspace)


def mla_append_decode_split(q_nope, q_pe, c_new, pe_new, latent_pages, page_table,
                            len_in, len_out, scale, max_len, n_workgroups=0,
                            workspace=None):
    """Deferred-combine absorbed-MLA step (ws_mla_append_decode_split);
    finish with merge_split.  Returns a SplitStep."""
    dev = latent_pages.device
    _require(q_nope, "q_nope", torch.bfloat16, dev, 2)
    _require(q_pe, "q_pe", torch.bfloat16, dev, 2)
    _require(latent_pages, "latent_pages", torch.bfloat16, dev, 3)
    _require(page_table, "page_table", torch.int32, dev, 2)
    _require(len_in, "len_in", torch.int32, dev, 1)
    _require(len_out, "len_out", torch.int32, dev, 1)
    B = page_table.shape[0]
    for t, n, w in ((c_new, "c_new", MLA_C), (pe_new, "pe_new", MLA_PE)):
        _require(t, n, torch.bfloat16, dev, 3, contiguous=False)
        if t.shape != (B, 1, w) or t.stride(2) != 1:
            raise ValueError(f"{n} must be [B, 1, {w}] with unit last stride")
    P, PS, L = latent_pages.shape
    rows = q_nope.shape[0]
    if L != MLA_LATENT or q_nope.shape[1] != MLA_C or q_pe.shape != (rows, MLA_PE):
        raise ValueError("MLA layout is q_nope 512 + q_pe 64 over a 576 latent")
    if B == 0 or rows % B or len_in.shape[0] != B or len_out.shape[0] != B:
        raise ValueError("rows must be B * H with B = page_table.shape[0]")
    if len_out.data_ptr() == len_in.data_ptr():
        raise ValueError("len_out must be a separate [B] int32 tensor")
    H = rows // B
    out = torch.empty((rows, MLA_C), dtype=torch.float32, device=dev)
    lse = torch.empty((rows,), dtype=torch.float32, device=dev)
    nwg, wsb = decode_plan(1, B, H, int(max_len), int(n_workgroups))
    if workspace is None:
        workspace = torch.zeros(max(wsb, 256), dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < wsb:
        raise ValueError(f"workspace needs {wsb} bytes")
    return _mla_split_launch(q_nope, q_pe, c_new, pe_new, latent_pages, page_table, len_in,
                             len_out, scale, max_len, nwg, out, lse, workspace)


def _mla_split_launch(q_nope, q_pe, c_new, pe_new, latent_pages, page_table, len_in, len_out,
                      scale, max_len, nwg, out, lse, workspace) -> SplitStep:
    """The ws_mla_append_decode_split launch on arguments already checked
    (mla_append_decode_split, or a cache that owns the pools, page table,
    lengths, partial buffers and workspace); returns the SplitStep."""
    B = page_table.shape[0]
    P, PS, _ = latent_pages.shape
    H = q_nope.shape[0] // B
    _check(lib().ws_mla_append_decode_split(
        _ptr(q_nope), _ptr(q_pe), _ptr(c_new), c_new.stride(0), _ptr(pe_new),
        pe_new.stride(0), _ptr(latent_pages), _ptr(page_table), _ptr(len_in),
        _ptr(len_out), B, H, PS, page_table.shape[1], P, int(max_len), nwg, float(scale),
        _ptr(out), _ptr(lse), _ptr(workspace), workspace.numel() * workspace.element_size(),
        _stream(latent_pages.device)), "ws_mla_append_decode_split")
    return SplitStep(len_out, B, 1, H, MLA_C, PS * page_table.shape[1], nwg, out, lse,
                     workspace)


def merge_split(step: SplitStep, b=None, fmt=PARTIAL_LSE_F32, out_dtype=torch.bfloat16,
                want_lse=True, out=None, lse_out=None):
    """Finish a deferred-combine step (ws_merge_split): combine its GPU pieces
    with the host partial `b` (formats as lse_merge; None = no host partial),
    normalise.  Returns (out [rows, Dv] in out_dtype, lse [rows] or None)."""
    step.check_workspace()
    dev = step.out_g.device
    rows = step.out_g.numel() // step.Dv
    b_out, b_aux0, b_aux1 = _host_operand(b, fmt, rows, step.Dv, dev)
    if out is None:
        out = torch.empty((rows, step.Dv), dtype=out_dtype, device=dev)
    if want_lse and lse_out is None:
        lse_out = torch.empty((rows,), dtype=torch.float32, device=dev)
    o16, o32 = (out, None) if out.dtype == torch.bfloat16 else (None, out)
    if out.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("merged output must be bfloat16 or float32")
    ws = step.workspace
    _check(lib().ws_merge_split(
        _ptr(step.gpu_len), step.B, step.rows_per_seq, step.heads, step.Dv, step.cap,
        step.nwg, _ptr(step.out_g), _ptr(step.lse_g), _ptr(ws), ws.numel() * ws.element_size(),
        _ptr(b_out), _ptr(b_aux0), _ptr(b_aux1), int(fmt), _ptr(o16), _ptr(o32),
        _ptr(lse_out if want_lse else None), _stream(dev)), "ws_merge_split")
    return out, (lse_out if want_lse else None)


def _require_operand(t, name, dtype, dev):
    """A merge's host operand: a tensor on `dev`, or a pinned host tensor,
    which the merge kernel reads in place over the host link."""
    if isinstance(t, torch.Tensor) and not t.is_cuda:
        if not t.is_pinned():
            raise ValueError(f"{name} must be on {dev} or in pinned host memory")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return
    _require(t, name, dtype, dev)


def _host_operand(b, fmt, rows, Dv, dev):
    """Pointers of the host partial `b` in format fmt (None: no host partial),
    validated against rows x Dv."""
    b_out = b_aux0 = b_aux1 = None
    if b is not None:
        if fmt in (PARTIAL_LSE_F32, PARTIAL_LSE_BF16):
            b_out, b_aux0 = b
            _require_operand(b_out, "b.out",
                             torch.float32 if fmt == PARTIAL_LSE_F32 else torch.bfloat16, dev)
            _require_operand(b_aux0, "b.lse", torch.float32, dev)
        elif fmt in (TRIPLE_UNNORM_F32, TRIPLE_NORM_BF16, TRIPLE_NORM_F32):
            b_out, b_aux0, b_aux1 = b
            dt = torch.bfloat16 if fmt == TRIPLE_NORM_BF16 else torch.float32
            _require_operand(b_out, "b.out", dt, dev)
            _require_operand(b_aux0, "b.max", dt, dev)
            _require_operand(b_aux1, "b.sum", dt, dev)
            if b_aux1.numel() != rows:
                raise ValueError("b.sum must have one value per row")
        else:
            raise ValueError(f"unknown host-partial format {fmt}")
        if b_out.numel() != rows * Dv or b_aux0.numel() != rows:
            raise ValueError("host partial does not match the step's rows")
    return b_out, b_aux0, b_aux1


def merge_split_uv(step: SplitStep, w_uv: torch.Tensor, b=None, fmt=PARTIAL_LSE_F32,
                   want_latent=False, want_lse=False):
    """Finish an absorbed-MLA split step with the W_UV epilogue
    (ws_mla_merge_split_uv): w_uv [heads, Dout, 512] bf16.  Returns
    (out_v [B, heads * Dout] bf16, latent [B * heads, 512] bf16 or None,
    lse [B * heads] or None)."""
    step.check_workspace()
    dev = step.out_g.device
    if step.rows_per_seq != 1 or step.Dv != MLA_C:
        raise ValueError("merge_split_uv finishes an MLA step")
    H = step.heads
    _require(w_uv, "w_uv", torch.bfloat16, dev, 3)
    if w_uv.shape[0] != H or w_uv.shape[2] != MLA_C:
        raise ValueError(f"w_uv must be [{H}, Dout, {MLA_C}]")
    Dout = w_uv.shape[1]
    rows = step.B * H
    b_out, b_aux0, b_aux1 = _host_operand(b, fmt, rows, MLA_C, dev)
    out_v = torch.empty((step.B, H * Dout), dtype=torch.bfloat16, device=dev)
    latent = (torch.empty((rows, MLA_C), dtype=torch.bfloat16, device=dev)
              if want_latent else None)
    lse = torch.empty((rows,), dtype=torch.float32, device=dev) if want_lse else None
    ws = step.workspace
    _check(lib().ws_mla_merge_split_uv(
        _ptr(step.gpu_len), step.B, H, step.cap, step.nwg, _ptr(step.out_g), _ptr(step.lse_g),
        _ptr(ws), ws.numel() * ws.element_size(), _ptr(b_out), _ptr(b_aux0), _ptr(b_aux1),
        int(fmt), _ptr(w_uv), Dout, _ptr(latent), _ptr(out_v), _ptr(lse), _stream(dev)),
        "ws_mla_merge_split_uv")
    return out_v, latent, lse


def split_reduce(part_out, part_lse, gpu_len, heads_per_len, tokens_per_split,
                 out=None, lse=None):
    """LSE-combine split partials part_out [n_splits, rows, Dv],
    part_lse [n_splits, rows] (see ws_split_reduce)."""
    dev = part_out.device
    _require(part_out, "part_out", torch.float32, dev, 3)
    _require(part_lse, "part_lse", torch.float32, dev, 2)
    _require(gpu_len, "gpu_len", torch.int32, dev, 1)
    ns, rows, Dv = part_out.shape
    if out is None:
        out = torch.empty((rows, Dv), dtype=torch.float32, device=dev)
    if lse is None:
        lse = torch.empty((rows,), dtype=torch.float32, device=dev)
    _check(lib().ws_split_reduce(_ptr(part_out), _ptr(part_lse), _ptr(gpu_len), rows,
                                 int(heads_per_len), Dv, ns, int(tokens_per_split),
                                 _ptr(out), _ptr(lse), _stream(dev)), "ws_split_reduce")
    return out, lse


# ---------------------------------------------------------------------------
# merge


def lse_merge(out_g, lse_g, b, fmt=PARTIAL_LSE_F32, out_dtype=torch.bfloat16,
              want_lse=True, out=None, lse_out=None):
    """Merge the GPU partial (out_g [..., Dv] fp32, lse_g [...] fp32) with a
    second partial `b`:
      fmt PARTIAL_LSE_F32   b = (out fp32, lse fp32)
      fmt TRIPLE_UNNORM_F32 b = (o unnormalised fp32, max fp32, sum fp32)
      fmt TRIPLE_NORM_BF16  b = (out bf16 normalised, max bf16, sum bf16)
      fmt TRIPLE_NORM_F32   b = (out fp32 normalised, max fp32, sum fp32)
      fmt PARTIAL_LSE_BF16  b = (out bf16 normalised, lse fp32)
    Returns (merged out in out_dtype (bf16 or fp32), lse fp32 or None)."""
    dev = out_g.device
    _require(out_g, "out_g", torch.float32, dev)
    _require(lse_g, "lse_g", torch.float32, dev)
    Dv = out_g.shape[-1]
    rows = out_g.numel() // Dv
    if lse_g.numel() != rows:
        raise ValueError("lse_g must have one value per output row")
    if b is None:
        raise ValueError("lse_merge needs a second partial")
    b_out, b_aux0, b_aux1 = _host_operand(b, fmt, rows, Dv, dev)
    if out is None:
        out = torch.empty(out_g.shape, dtype=out_dtype, device=dev)
    if want_lse and lse_out is None:
        lse_out = torch.empty(lse_g.shape, dtype=torch.float32, device=dev)
    if out.dtype == torch.bfloat16:
        o16, o32 = out, None
    elif out.dtype == torch.float32:
        o16, o32 = None, out
    else:
        raise TypeError("merged output must be bfloat16 or float32")
    _require(out, "out", out.dtype, dev)
    _check(lib().ws_lse_merge(_ptr(out_g), _ptr(lse_g), _ptr(b_out), _ptr(b_aux0),
                              _ptr(b_aux1), int(fmt), _ptr(o16), _ptr(o32),
                              _ptr(lse_out if want_lse else None), rows, Dv,
                              _stream(dev)), "ws_lse_merge")
    return out, (lse_out if want_lse else None)


# ---------------------------------------------------------------------------
# a request's path into the pages: pages and slots, rotary positions with the
# write, decode over 8-bit pages, prompt attention

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def _run(name: str, dev: torch.device, *args) -> None:
    """The entry point `name` on the current stream of `dev`, with `dev` the
    current device for the launch (the operands may live on another one than
    the caller's current)."""
    fn = getattr(lib(), name)
    if torch._C._cuda_getDevice() == dev.index:
        _check(fn(*args, _stream(dev)), name)
    else:
        with torch.cuda.device(dev):
            _check(fn(*args, _stream(dev)), name)


def _gpu(t, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (got {t.device})")
    return t.device


def _require_all(dev, specs, tensors) -> None:
    """_require of every (name, dtype, dims) of specs, in one pass while all is well."""
    idx = dev.index
    for (_, dtype, ndim), t in zip(specs, tensors):
        if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == idx
                and t.dim() == ndim and t.is_contiguous()):
            break
    else:
        return
    for (name, dtype, ndim), t in zip(specs, tensors):
        _require(t, name, dtype, dev, ndim)


_EXTEND_ARGS = (("page_table", torch.int32, 2), ("len_in", torch.int32, 1), ("n_new", torch.int32, 1),
                ("stack", torch.int32, 1), ("free_in", torch.int32, 1))
_RELEASE_ARGS = (("page_table", torch.int32, 2), ("len_in", torch.int32, 1), ("done", torch.bool, 1),
                 ("stack", torch.int32, 1), ("free_in", torch.int32, 1))
_POOL_ARGS = {bits: (("k_pages", dt, 4), ("v_pages", dt, 4)) for bits, dt in
              ((16, torch.bfloat16), (8, E4M3))}
_SCALE_ARGS = (("k_scale", E8M0, 3), ("v_scale", E8M0, 3))
_DECODE16_ARGS = (("q", torch.bfloat16, 3), ("k_pages", torch.bfloat16, 4), ("v_pages", torch.bfloat16, 4),
                  ("page_table", torch.int32, 2), ("gpu_len", torch.int32, 1))
_DECODE8_ARGS = (("q", torch.bfloat16, 3), ("page_table", torch.int32, 2), ("gpu_len", torch.int32, 1))
_PROMPT_ARGS = (("q", torch.bfloat16, 3), ("page_table", torch.int32, 2), ("kv_len", torch.int32, 1),
                ("cu_new", torch.int32, 1))


class PageStep(NamedTuple):
    """What pages_extend hands out (all int32 on the GPU)."""

    len_out: torch.Tensor    # [B] lengths with the new tokens; -1 where they got no place
    cu_new: torch.Tensor     # [B + 1] each sequence's first token of the packed batch
    positions: torch.Tensor  # [n_tokens]
    slots: torch.Tensor      # [n_tokens] page * page_size + offset, or -1
    free_out: torch.Tensor   # [1] free pages left on the stack


def pages_extend(page_table, len_in, n_new, stack, free_in, page_size, num_pages, n_tokens,
                 pos_base=None) -> PageStep:
    """Pages and slots for n_new[b] more tokens of every sequence, from the
    stack of free pages stack[:free_in] (ws_pages_extend): new page ids go into
    page_table in place, everything else into new tensors, so a call that is
    not wanted is undone by keeping len_in and free_in.  n_tokens: the packed
    batch's tokens, sum(n_new) or more (the rest is padding: slot -1).
    pos_base [B]: what a position counts beside the partition's tokens."""
    dev = _gpu(page_table, "page_table")
    _require_all(dev, _EXTEND_ARGS, (page_table, len_in, n_new, stack, free_in))
    B, max_pages = page_table.shape
    N = int(n_tokens)
    if len_in.shape[0] != B or n_new.shape[0] != B or free_in.shape[0] != 1:
        raise ValueError("len_in and n_new must be [B] and free_in [1]")
    if pos_base is not None:
        _require(pos_base, "pos_base", torch.int32, dev, 1)
        if pos_base.shape[0] != B:
            raise ValueError("pos_base must be [B]")
    if N < 0:
        raise ValueError(f"n_tokens {N} < 0")
    buf = torch.empty(2 * B + 2 + 2 * N, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    _run("ws_pages_extend", dev, page_table.data_ptr(), len_in.data_ptr(), n_new.data_ptr(),
         stack.data_ptr(), free_in.data_ptr(), _ptr(pos_base), at, at + 4 * B, at + 8 * B + 4,
         at + 8 * B + 4 + 4 * N, at + 8 * B + 4 + 8 * N, B, max_pages, int(num_pages),
         stack.shape[0], int(page_size), N)
    return PageStep(*buf.split_with_sizes((B, B + 1, N, N, 1)))


def pages_release(page_table, len_in, done, stack, free_in, page_size):
    """The pages of the sequences with done[b] (bool [B]) back on the stack, in
    place (ws_pages_release).  Returns (lengths: 0 for those, free pages)."""
    dev = _gpu(page_table, "page_table")
    _require_all(dev, _RELEASE_ARGS, (page_table, len_in, done, stack, free_in))
    B, max_pages = page_table.shape
    if len_in.shape[0] != B or done.shape[0] != B or free_in.shape[0] != 1:
        raise ValueError("len_in and done must be [B] and free_in [1]")
    buf = torch.empty(B + 1, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    _run("ws_pages_release", dev, page_table.data_ptr(), len_in.data_ptr(), done.data_ptr(),
         stack.data_ptr(), free_in.data_ptr(), at, at + 4 * B, B, max_pages, stack.shape[0],
         int(page_size))
    return buf.split_with_sizes((B, 1))


@functools.lru_cache(maxsize=256)
def _axis_bytes(pair_axis: tuple) -> bytes:
    if any(a != int(a) or not 0 <= a < 4 for a in pair_axis):
        raise ValueError("pair_axis must hold axis numbers from 0 to 3")
    return bytes(int(a) for a in pair_axis)


def rope_sections(sections, interleaved=False) -> list:
    """pair_axis of sections[a] pairs on axis a: one axis after the other, or
    interleaved (0 1 2 0 1 2 ..., an axis dropping out once its pairs are used)."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a] > 0:
                left[a] -= 1
                out.append(a)
    return out


def _rope_rows(t, name, dev, N=None, D=None):
    """(heads, token stride) of a [N, heads, D] bf16 operand whose tokens may be
    strided (a slice of a fused projection's rows)."""
    if (isinstance(t, torch.Tensor) and t.dtype is torch.bfloat16 and t.get_device() == dev.index
            and t.dim() == 3):  # (as below, in one pass while all is well)
        n, heads, d = t.shape
        st, sh, sd = t.stride()
        if n and heads and sd == 1 and sh == d and (N is None or n == N) and (D is None or d == D):
            return heads, (st if n > 1 else heads * d)
    _require(t, name, torch.bfloat16, dev, 3, contiguous=False)
    n, heads, d = t.shape
    if (N is not None and n != N) or (D is not None and d != D):
        raise ValueError(f"{name} must be [{N}, heads, {D}] (got {tuple(t.shape)})")
    if heads == 0 or (n > 0 and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != d))):
        raise ValueError(f"{name} must have contiguous [heads, D] rows (strides {t.stride()})")
    return heads, (t.stride(0) if n > 1 else heads * d)


def _rope_args(q, k, positions, inv_freq, pair_axis, dev):
    Hq, q_stride = _rope_rows(q, "q", dev)
    N, _, D = q.shape
    Hkv, k_stride = _rope_rows(k, "k", dev, N, D)
    _require(positions, "positions", torch.int32, dev)
    _require(inv_freq, "inv_freq", torch.float32, dev, 1)
    shape = positions.shape
    if len(shape) not in (1, 2) or shape[-1] != N:
        raise ValueError(f"positions must be [N] or [axes, N], N = {N} (got {tuple(shape)})")
    axes = shape[0] if len(shape) == 2 else 1
    half = inv_freq.shape[0]
    axis = None
    if pair_axis is not None:
        axis = _axis_bytes(tuple(pair_axis))
        if len(axis) != half:
            raise ValueError(f"pair_axis has {len(axis)} pairs, inv_freq {half}")
    return N, Hq, Hkv, D, q_stride, k_stride, axes, axis, 2 * half


def rope(q, k, positions, inv_freq, pair_axis=None, adjacent=False, factor=1.0, q_out=None,
         k_out=None):
    """Rotary positions of q [N, Hq, D] and k [N, Hkv, D] (ws_rope; tokens may be
    strided).  positions [N] or [axes, N] int32; inv_freq [rot / 2] fp32, the
    radians a position turns each pair; pair_axis: the axis of each pair
    (rope_sections; None: axis 0); adjacent: pairs (2 i, 2 i + 1) instead of
    (i, i + rot / 2); factor scales the rotated columns.  Returns contiguous
    (q_out, k_out)."""
    dev = _gpu(q, "q")
    N, Hq, Hkv, D, qs, ks, axes, axis, rot = _rope_args(q, k, positions, inv_freq, pair_axis, dev)
    if q_out is None:
        q_out = q.new_empty((N, Hq, D))
    else:
        _require(q_out, "q_out", torch.bfloat16, dev, 3)
    if k_out is None:
        k_out = k.new_empty((N, Hkv, D))
    else:
        _require(k_out, "k_out", torch.bfloat16, dev, 3)
    if q_out.shape != q.shape or k_out.shape != k.shape:
        raise ValueError("q_out and k_out must have q's and k's shapes")
    if N == 0:
        return q_out, k_out
    _run("ws_rope", dev, _ptr(q), qs, _ptr(k), ks, _ptr(positions), axes, _ptr(inv_freq), axis,
         int(bool(adjacent)), float(factor), _ptr(q_out), _ptr(k_out), N, Hq, Hkv, D, rot)
    return q_out, k_out


def _pools(k_pages, v_pages, k_scale, v_scale, dev):
    """(num_pages, Hkv, page_size, D) of bf16 pools, or of 8-bit ones with scales."""
    shape = k_pages.shape
    if k_scale is None and v_scale is None:
        _require_all(dev, _POOL_ARGS[16], (k_pages, v_pages))
    else:
        if k_scale is None or v_scale is None:
            raise ValueError("8-bit pools take both k_scale and v_scale")
        _require_all(dev, _POOL_ARGS[8], (k_pages, v_pages))
        _require_all(dev, _SCALE_ARGS, (k_scale, v_scale))
        if k_scale.shape != shape[:3] or v_scale.shape != k_scale.shape:
            raise ValueError("k_scale and v_scale must be [num_pages, Hkv, page_size]")
    if v_pages.shape != shape:
        raise ValueError("k/v page pools differ in shape")
    return shape


def rope_append(q, k, v, positions, inv_freq, slots, k_pages, v_pages, k_scale=None, v_scale=None,
                pair_axis=None, adjacent=False, factor=1.0, q_out=None):
    """rope() of q, and of k into the pages with v beside it (ws_rope_append):
    token t's keys and values go to slot slots[t] (pages_extend) of the pools,
    bf16, or e4m3 with k_scale and v_scale (one power of two per token and KV
    head).  A slot outside the pools (-1) writes nothing; slots must differ.
    Returns q_out [N, Hq, D]."""
    dev = _gpu(q, "q")
    N, Hq, Hkv, D, qs, ks, axes, axis, rot = _rope_args(q, k, positions, inv_freq, pair_axis, dev)
    Hv, vs = _rope_rows(v, "v", dev, N, D)
    _require(slots, "slots", torch.int32, dev, 1)
    P, Hp, PS, Dp = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    if Hv != Hkv or Hp != Hkv or Dp != D or slots.shape[0] != N:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}, slots {tuple(slots.shape)} and pools "
                         f"{tuple(k_pages.shape)} do not match")
    if q_out is None:
        q_out = q.new_empty((N, Hq, D))
    else:
        _require(q_out, "q_out", torch.bfloat16, dev, 3)
        if q_out.shape != q.shape:
            raise ValueError("q_out must have q's shape")
    if N == 0:
        return q_out
    _run("ws_rope_append", dev, _ptr(q), qs, _ptr(k), ks, _ptr(v), vs, _ptr(positions), axes,
         _ptr(inv_freq), axis, int(bool(adjacent)), float(factor), _ptr(slots), _ptr(q_out),
         _ptr(k_pages), _ptr(v_pages), _ptr(k_scale), _ptr(v_scale), N, Hq, Hkv, D, rot, PS, P)
    return q_out


def gqa8_plan(rows_kv: int, heads: int, D: int, max_len: int, n_workgroups: int = 0):
    """(n_splits, workspace_bytes) of a decode call over 8-bit pages."""
    key = ("gqa8", rows_kv, heads, D, max_len, n_workgroups,
           torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -1)
    hit = _plans.get(key)
    if hit is not None:
        return hit
    n, wsb = ctypes.c_int(0), ctypes.c_size_t(0)
    _check(lib().ws_gqa8_decode_plan(rows_kv, heads, D, max_len, n_workgroups, ctypes.byref(n),
                                     ctypes.byref(wsb)), "ws_gqa8_decode_plan")
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = (n.value, wsb.value)
    return n.value, wsb.value


def _gqa8_decode(name, q, k_pages, v_pages, k_scale, v_scale, page_table, gpu_len, scale, max_len,
                 n_workgroups, out_bf16, out, lse):
    dev = _gpu(k_pages, "k_pages")
    if k_scale is None or v_scale is None:
        raise ValueError("8-bit pools take both k_scale and v_scale")
    P, Hkv, PS, D = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    _require_all(dev, _DECODE8_ARGS, (q, page_table, gpu_len))
    B, Hq, Dq = q.shape
    if Dq != D or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match the pools {tuple(k_pages.shape)}")
    if page_table.shape[0] != B or gpu_len.shape[0] != B:
        raise ValueError("page_table/gpu_len batch mismatch")
    if lse is None:
        lse = torch.empty((B, Hq), dtype=torch.float32, device=dev)
    else:
        _require(lse, "lse", torch.float32, dev, 2)
        if lse.shape != (B, Hq):
            raise ValueError("lse must be [B, Hq]")
    if out is not None:
        _require(out, "out", torch.float32, dev, 3)
        if out.shape != q.shape:
            raise ValueError("out must be [B, Hq, D]")
    elif out_bf16 is None:
        out = torch.empty((B, Hq, D), dtype=torch.float32, device=dev)
    if B == 0:
        return out, lse
    nwg, wsb = gqa8_plan(B * Hkv, Hq // Hkv, D, int(max_len), int(n_workgroups))
    # the call's own: a buffer kept between calls would be shared by graphs that
    # were captured one after the other and replay together
    wsb = (wsb + 255) & ~255
    if out_bf16 is None:
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        outs = (out.data_ptr(), lse.data_ptr(), ws.data_ptr())
    else:  # the fp32 output, which the merge rounds, lies behind the pieces
        ws = torch.empty(wsb + 4 * B * Hq * D, dtype=torch.uint8, device=dev)
        outs = (out_bf16.data_ptr(), ws.data_ptr() + wsb, lse.data_ptr(), ws.data_ptr())
    _run(name, dev, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(),
         v_scale.data_ptr(), page_table.data_ptr(), gpu_len.data_ptr(), B, Hq, Hkv, D, PS,
         page_table.shape[1], P, int(max_len), nwg, float(scale), *outs, wsb)
    return out, lse


def gqa8_decode_partial(q, k_pages, v_pages, k_scale, v_scale, page_table, gpu_len, scale, max_len,
                        n_workgroups=0, out=None, lse=None):
    """gqa_decode_partial over 8-bit pages (ws_gqa8_decode_partial): q [B, Hq, D]
    bf16, pools [P, Hkv, PS, D] float8_e4m3fn with scales [P, Hkv, PS]
    float8_e8m0fnu -> (out [B, Hq, D] fp32 normalised, lse [B, Hq] fp32).
    max_len must bound every gpu_len[b]."""
    return _gqa8_decode("ws_gqa8_decode_partial", q, k_pages, v_pages, k_scale, v_scale, page_table,
                        gpu_len, scale, max_len, n_workgroups, None, out, lse)


def gqa8_decode_full(q, k_pages, v_pages, k_scale, v_scale, page_table, gpu_len, scale, max_len,
                     n_workgroups=0, out_bf16=None, lse=None):
    """gqa8_decode_partial for a partition that holds every token: returns
    (out [B, Hq, D] bf16, lse [B, Hq] fp32)."""
    dev = _gpu(q, "q")
    if out_bf16 is None:
        _require(q, "q", torch.bfloat16, dev, 3)
        out_bf16 = torch.empty_like(q)
    else:
        _require(out_bf16, "out_bf16", torch.bfloat16, dev, 3)
        if out_bf16.shape != q.shape:
            raise ValueError("out_bf16 must have q's shape")
    _, lse = _gqa8_decode("ws_gqa8_decode_full", q, k_pages, v_pages, k_scale, v_scale, page_table,
                          gpu_len, scale, max_len, n_workgroups, out_bf16, None, lse)
    return out_bf16, lse


def gqa_prompt_plan(n_tokens: int, batch: int, Hq: int, Hkv: int, D: int, max_len: int,
                    n_splits: int = 0, fp8: bool = False):
    """(pieces, workspace_bytes) of a prompt call: how many pieces its split tiles
    can leave (0: no tile is split, no workspace)."""
    key = ("prompt", n_tokens, batch, Hq, Hkv, D, max_len, n_splits, fp8,
           torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -1)
    hit = _plans.get(key)
    if hit is not None:
        return hit
    n, wsb = ctypes.c_int(0), ctypes.c_size_t(0)
    _check(lib().ws_gqa_prompt_plan(n_tokens, batch, Hq, Hkv, D, int(fp8), max_len, n_splits,
                                    ctypes.byref(n), ctypes.byref(wsb)), "ws_gqa_prompt_plan")
    if len(_plans) > 4096:
        _plans.clear()
    _plans[key] = (n.value, wsb.value)
    return n.value, wsb.value


def gqa_prompt(q, k_pages, v_pages, page_table, kv_len, cu_new, scale, max_len, k_scale=None,
               v_scale=None, n_splits=0, out_dtype=torch.bfloat16, want_lse=True, out=None, lse=None):
    """Causal attention of the new tokens of every sequence over the pages
    (ws_gqa_prompt): q [N, Hq, D] bf16, packed; sequence b's queries are rows
    cu_new[b] .. cu_new[b + 1] and the last of its kv_len[b] tokens in the pages.
    Pools bf16, or 8-bit with k_scale and v_scale.  Returns (out [N, Hq, D] in
    out_dtype (bf16 or fp32), lse [N, Hq] fp32 or None); rows outside
    [cu_new[0], cu_new[B]) are not written.  max_len must bound every kv_len[b].
    n_splits: workgroups that share a tile of rows (0: the library's choice by
    the lengths)."""
    dev = _gpu(k_pages, "k_pages")
    P, Hkv, PS, D = _pools(k_pages, v_pages, k_scale, v_scale, dev)
    _require_all(dev, _PROMPT_ARGS, (q, page_table, kv_len, cu_new))
    N, Hq, Dq = q.shape
    B = page_table.shape[0]
    if Dq != D or Hkv == 0 or Hq % Hkv or Hq == 0:
        raise ValueError(f"q {tuple(q.shape)} does not match the pools {tuple(k_pages.shape)}")
    if kv_len.shape[0] != B or cu_new.shape[0] != B + 1:
        raise ValueError("kv_len must be [B] and cu_new [B + 1] for page_table's B rows")
    if out is None:
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("out_dtype must be bfloat16 or float32")
        out = torch.empty_like(q, dtype=out_dtype)
    else:
        if out.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError("out must be bfloat16 or float32")
        _require(out, "out", out.dtype, dev, 3)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
    if lse is not None:
        _require(lse, "lse", torch.float32, dev, 2)
        if lse.shape != (N, Hq):
            raise ValueError("lse must be [N, Hq]")
    elif want_lse:
        lse = torch.empty((N, Hq), dtype=torch.float32, device=dev)
    if N == 0 or B == 0:
        return out, lse
    _, wsb = gqa_prompt_plan(N, B, Hq, Hkv, D, int(max_len), int(n_splits), k_scale is not None)
    ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
    o16, o32 = (out, None) if out.dtype == torch.bfloat16 else (None, out)
    _run("ws_gqa_prompt", dev, _ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(k_scale), _ptr(v_scale),
         _ptr(page_table), _ptr(kv_len), _ptr(cu_new), N, B, Hq, Hkv, D, PS, page_table.shape[1], P,
         int(max_len), int(n_splits), float(scale), _ptr(o16), _ptr(o32), _ptr(lse), _ptr(ws), wsb)
    return out, lse
