"""Serving ops over a paged KV cache, for batches of sequences of any lengths.

A cache is two pools of pages, `k_pages` and `v_pages` [n_pages, n_kv, page_size, head_dim] (fp16 or bf16), and an
int32 `page_table` [B, width] whose row b lists the pages of sequence b in order. `lengths` (int32 [B]) counts
each sequence's positions including the call's own tokens; `starts` (int32 [B + 1]) gives the token rows
starts[b]..starts[b+1] of sequence b, its last positions, or None: one token per sequence. All of them live on the
device and are read there, so a captured call serves every step. A length <= 0 marks an unused slot of the batch.

`paged_append` rotates q and k by their positions and writes k and v into the pages; `paged_attention` attends
causally over the pages, optionally limited to a sliding window and a few first tokens (sinks);
`shared_prefix_attention` attends over a prefix that all sequences share, read once for all of them, and over
each sequence's own pages. The reference keeps one contiguous cache per sequence and one position for the whole batch
(kernels/e2e/model.py:192, 236-244); these ops have no counterpart there.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from kernels import _lib

MAX_GROUP = 16  # query heads per kv head
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, tokens):
    """(n_pages, n_kv, page_size, head_dim, B) of a checked cache and batch."""
    need = _lib.require_extent
    need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape,
         f"{what}: k_pages and v_pages must be [n_pages, n_kv, page_size, head_dim], both alike")
    need(k_pages.is_contiguous() and v_pages.is_contiguous(), f"{what}: pages must be contiguous")
    n_pages, n_kv, page, hd = k_pages.shape
    need(n_pages > 0 and n_kv > 0, f"{what}: an empty pool of pages")
    need(16 <= page <= 256 and page & (page - 1) == 0, f"{what}: page_size must be a power of two from 16 to 256")
    need(hd == 64 or hd == 128, f"{what}: head_dim must be 64 or 128")
    need(page_table.dim() == 2 and page_table.shape[1] > 0 and page_table.stride(1) == 1,
         f"{what}: page_table must be [sequences, pages] with unit column stride")
    B = page_table.shape[0]
    need(lengths.dim() == 1 and lengths.shape[0] == B and lengths.is_contiguous(),
         f"{what}: lengths must hold one count per row of page_table")
    if starts is None:
        need(tokens == B, f"{what}: without starts there is one token per sequence")
    else:
        need(starts.dim() == 1 and starts.shape[0] == B + 1 and starts.is_contiguous(),
             f"{what}: starts must hold sequences + 1 row numbers")
    if not (page_table.dtype == lengths.dtype == torch.int32 and (starts is None or starts.dtype == torch.int32)):
        raise RuntimeError(f"{what}: page_table, lengths and starts must be int32")
    if k_pages.dtype not in _DTYPES or v_pages.dtype != k_pages.dtype:
        raise RuntimeError(f"{what}: pages must be fp16 or bf16, both alike")
    return n_pages, n_kv, page, hd, B


def _on_one_device(what, *tensors):
    device = tensors[0].device
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                raise RuntimeError(f"{what}: tensors must be on a CUDA device (no CPU path), got {t.device}")
            if t.device != device:
                raise RuntimeError(f"{what}: tensors on {device} and {t.device}")


def paged_append(qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts=None, offset=0, out=None):
    """Rotate q and k of qkv [T, (n_heads + 2 n_kv) * head_dim] (q heads, k heads, v heads; unit column stride) by
    their tokens' positions and append k and v to the pages, in place. cos, sin [positions, head_dim / 2]: one angle
    per pair of dims d, d + head_dim / 2, fp32 or qkv's type, rows taken at the own position + offset (the length
    of a shared prefix). The rotation is computed in fp32 and rounded once. Returns the rotated q [T, n_heads,
    head_dim] (`out` if given). A token without a page, or past the tables, appends nothing and sets the device error
    DK_DEVERR_BAD_POSITION; one of an unused slot appends nothing and returns zeros."""
    what = "paged_append"
    _lib.require_extent(qkv.dim() == 2, f"{what}: qkv must be [tokens, (n_heads + 2 n_kv) * head_dim]")
    T = qkv.shape[0]
    n_pages, kv, page, hd, B = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, T)
    _lib.require_extent(n_kv == kv and n_heads > 0 and qkv.shape[1] == (n_heads + 2 * n_kv) * hd and qkv.stride(1) == 1,
                        f"{what}: qkv must be [tokens, (n_heads + 2 n_kv) * head_dim] with the pages' kv heads")
    _lib.require_extent(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == hd // 2 and cos.stride(1) == 1
                        and cos.stride() == sin.stride(), f"{what}: cos and sin must be [positions, head_dim / 2]")
    _lib.require_extent(offset >= 0, f"{what}: offset must not be negative")
    if qkv.dtype != k_pages.dtype:
        raise RuntimeError(f"{what}: qkv is {qkv.dtype}, the pages are {k_pages.dtype}")
    if cos.dtype != sin.dtype or (cos.dtype != torch.float32 and cos.dtype != qkv.dtype):
        raise RuntimeError(f"{what}: cos and sin must be fp32 or qkv's type")
    if out is not None:
        _lib.require_extent(tuple(out.shape) == (T, n_heads, hd) and out.is_contiguous() and out.dtype == qkv.dtype,
                            f"{what}: out must be a contiguous [tokens, n_heads, head_dim] of qkv's type")
    _on_one_device(what, qkv, k_pages, v_pages, page_table, lengths, starts, cos, sin, out)
    q = torch.empty((T, n_heads, hd), dtype=qkv.dtype, device=qkv.device) if out is None else out
    _lib.call("dk_paged_append", qkv.data_ptr(), qkv.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page,
              page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
              None if starts is None else starts.data_ptr(), cos.data_ptr(), sin.data_ptr(),
              1 if cos.dtype == torch.float32 else 0, cos.stride(0), cos.shape[0], offset, q.data_ptr(), T, B, n_heads,
              n_kv, hd, _DTYPES[qkv.dtype], torch.cuda.current_stream(qkv.device).cuda_stream)
    return q


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(T, B, nq, nkv, hd, dtype, ragged, prefix, device):
    n = ctypes.c_uint64(0)
    with torch.cuda.device(device):
        _lib.call("dk_paged_attention_workspace_bytes", T, B, nq, nkv, hd, dtype, ragged, prefix, ctypes.byref(n))
    return int(n.value)


def _check_queries(what, q, k_pages, n_kv, hd, scale, out):
    _lib.require_extent(q.dim() == 3 and q.shape[2] == hd and q.stride(2) == 1 and q.stride(1) == hd,
                        f"{what}: q must be [tokens, heads, head_dim] with its heads side by side")
    nq = q.shape[1]
    _lib.require_extent(nq > 0 and nq % n_kv == 0 and nq // n_kv <= MAX_GROUP,
                        f"{what}: query heads must be a multiple of the kv heads, at most {MAX_GROUP} for each")
    if q.dtype != k_pages.dtype:
        raise RuntimeError(f"{what}: q is {q.dtype}, the pages are {k_pages.dtype}")
    if out is not None:
        _lib.require_extent(out.shape == q.shape and out.is_contiguous() and out.dtype == q.dtype,
                            f"{what}: out must be a contiguous tensor of q's shape and type")
    return hd ** -0.5 if scale is None else float(scale)


def paged_attention(q, k_pages, v_pages, page_table, lengths, starts=None, window=0, sinks=0, scale=None, out=None):
    """Attention of q [T, n_heads, head_dim] (tokens any stride apart) over the pages: the row at position p sees the
    positions j <= p of its sequence, with window > 0 only those with j > p - window or j < sinks. Returns [T,
    n_heads, head_dim] contiguous (`out` if given); a row that sees nothing is zero. scale: head_dim ** -0.5 if
    None. Pages that no row sees are not read, and their table entries may hold anything. With several tokens of a
    sequence in one call, the keys and values that one of them sees have to be finite for the others too."""
    what = "paged_attention"
    T = q.shape[0]
    n_pages, n_kv, page, hd, B = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, T)
    scale = _check_queries(what, q, k_pages, n_kv, hd, scale, out)
    _lib.require_extent(window >= 0 and sinks >= 0, f"{what}: window and sinks must not be negative")
    _on_one_device(what, q, k_pages, v_pages, page_table, lengths, starts, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nq, dtype = q.shape[1], _DTYPES[q.dtype]
    nbytes = _workspace_bytes(T, B, nq, n_kv, hd, dtype, starts is not None, 0, q.device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.call("dk_paged_attention", q.data_ptr(), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page,
              page_table.data_ptr(), page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
              None if starts is None else starts.data_ptr(), window, sinks, scale, out.data_ptr(), T, B, nq, n_kv, hd,
              dtype, ws.data_ptr(), nbytes, torch.cuda.current_stream(q.device).cuda_stream)
    return out


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, page_table, lengths, starts=None, scale=None,
                            out=None):
    """Attention of a batch whose sequences share a prefix: every row of q [T, n_heads, head_dim] sees the prefix's
    prefix_len positions (in the pages prefix_table lists, int32 [>= pages of the prefix]) and, causally, its own
    sequence's positions (page_table, lengths, starts: counted without the prefix). The prefix's keys and values are
    read once for all rows. Returns [T, n_heads, head_dim] (`out` if given)."""
    what = "shared_prefix_attention"
    if prefix_len == 0:
        return paged_attention(q, k_pages, v_pages, page_table, lengths, starts, scale=scale, out=out)
    T = q.shape[0]
    n_pages, n_kv, page, hd, B = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, T)
    scale = _check_queries(what, q, k_pages, n_kv, hd, scale, out)
    _lib.require_extent(prefix_len > 0 and prefix_table.dim() == 1 and prefix_table.is_contiguous()
                        and prefix_table.shape[0] >= math.ceil(prefix_len / page),
                        f"{what}: prefix_table must list the pages of prefix_len positions")
    if prefix_table.dtype != torch.int32:
        raise RuntimeError(f"{what}: prefix_table must be int32")
    _on_one_device(what, q, k_pages, v_pages, prefix_table, page_table, lengths, starts, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nq, dtype = q.shape[1], _DTYPES[q.dtype]
    nbytes = _workspace_bytes(T, B, nq, n_kv, hd, dtype, starts is not None, prefix_len, q.device)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.call("dk_shared_prefix_attention", q.data_ptr(), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), n_pages,
              page, prefix_table.data_ptr(), prefix_len, page_table.data_ptr(), page_table.stride(0),
              page_table.shape[1], lengths.data_ptr(), None if starts is None else starts.data_ptr(), scale,
              out.data_ptr(), T, B, nq, n_kv, hd, dtype, ws.data_ptr(), nbytes,
              torch.cuda.current_stream(q.device).cuda_stream)
    return out
