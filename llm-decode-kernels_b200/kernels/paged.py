"""Serving ops over a paged KV cache, for batches of sequences of any lengths.

A cache is two pools of pages, `k_pages` and `v_pages` [n_pages, n_kv, page_size, head_dim] (fp16 or bf16), and an
int32 `page_table` [B, width] whose row b lists the pages of sequence b in order. `lengths` (int32 [B]) counts
each sequence's positions including the call's own tokens; `starts` (int32 [B + 1]) gives the token rows
starts[b]..starts[b+1] of sequence b, its last positions, or None: one token per sequence. All of them live on the
device and are read there, so a captured call serves every step. A length <= 0 marks an unused slot of the batch; rows
before starts[0] and from starts[B] on belong to no sequence.

`paged_append` rotates q and k by their positions and writes k and v into the pages; `paged_attention` attends
causally over the pages, optionally limited to a sliding window and a few first tokens (sinks);
`shared_prefix_attention` attends over a prefix that all sequences share, read once for all of them, and over
each sequence's own pages. The reference keeps one contiguous cache per sequence and one position for the whole batch
(kernels/e2e/model.py:192, 236-244); these ops have no counterpart there.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from kernels import _lib

MAX_GROUP = 16  # query heads per kv head
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_INT32 = torch.int32
_raw_stream = torch._C._cuda_getCurrentRawStream  # (the public form builds a Stream object, about 1 us of each call)


# These calls are small next to their checks, so the checks are plain comparisons whose messages are only put together
# when one fails, and buffers come from the factory calls that take the least time (new_empty_strided 1.4 us, new_empty 1.8).
def _refuse(what: str, message: str):
    raise ValueError(f"{what}: {message}")


def _wrong_type(what: str, message: str):
    raise RuntimeError(f"{what}: {message}")


_FP4_ROWS = {72: 128, 36: 64}  # head_dim by the bytes of a position in a cache of 4-bit codes


def _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, tokens, fp4=False):
    """(n_pages, n_kv, page_size, head_dim, B, the table's row stride, its width) of a checked cache (fp4: of 4-bit codes,
    kernels.paged_fp4) and batch."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        _refuse(what, f"k_pages and v_pages must be [n_pages, n_kv, page_size, {'9/16 ' if fp4 else ''}head_dim], both alike")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        _refuse(what, "pages must be contiguous")
    n_pages, n_kv, page, hd = shape
    if fp4:
        hd = _FP4_ROWS.get(hd, 0)
    if n_pages <= 0 or n_kv <= 0:
        _refuse(what, "an empty pool of pages")
    if not (16 <= page <= 256 and page & (page - 1) == 0):
        _refuse(what, "page_size must be a power of two from 16 to 256")
    if hd != 128 and hd != 64:
        _refuse(what, "head_dim must be 64 or 128")
    if page_table.dim() != 2:
        _refuse(what, "page_table must be [sequences, pages] with unit column stride")
    B, table_width = page_table.shape
    ld_table, unit = page_table.stride()
    if table_width == 0 or unit != 1 and table_width > 1:
        _refuse(what, "page_table must be [sequences, pages] with unit column stride")
    if lengths.shape != (B,) or not lengths.is_contiguous():
        _refuse(what, "lengths must hold one count per row of page_table")
    if starts is None:
        if tokens != B:
            _refuse(what, "without starts there is one token per sequence")
    elif starts.shape != (B + 1,) or not starts.is_contiguous():
        _refuse(what, "starts must hold sequences + 1 row numbers")
    if not (page_table.dtype is _INT32 and lengths.dtype is _INT32 and (starts is None or starts.dtype is _INT32)):
        _wrong_type(what, "page_table, lengths and starts must be int32")
    if fp4:
        if k_pages.dtype is not torch.uint8 or v_pages.dtype is not torch.uint8:
            _wrong_type(what, "pages must be uint8, both of them")
    elif k_pages.dtype not in _DTYPES or v_pages.dtype is not k_pages.dtype:
        _wrong_type(what, "pages must be fp16 or bf16, both alike")
    return n_pages, n_kv, page, hd, B, ld_table, table_width


def paged_append(qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts=None, offset=0, out=None):
    """Rotate q and k of qkv [T, (n_heads + 2 n_kv) * head_dim] (q heads, k heads, v heads; unit column stride) by
    their tokens' positions and append k and v to the pages, in place. cos, sin [positions, head_dim / 2]: one angle
    per pair of dims d, d + head_dim / 2, fp32 or qkv's type, rows taken at the own position + offset (the length
    of a shared prefix). The rotation is computed in fp32 and rounded once. Returns the rotated q [T, n_heads,
    head_dim] (`out` if given). A token without a page, or past the tables, appends nothing and sets the device error
    DK_DEVERR_BAD_POSITION; one of an unused slot or of no sequence appends nothing and returns zeros."""
    return _append("paged_append", qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts, offset, out, None)


def _append(what, qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts, offset, out, scales):
    """`scales`: (k_scale, v_scale) of a cache of 4-bit codes, or None."""
    if qkv.dim() != 2:
        _refuse(what, "qkv must be [tokens, (n_heads + 2 n_kv) * head_dim]")
    T, width = qkv.shape
    n_pages, kv, page, hd, B, ld_table, table_width = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, T,
                                                                   scales is not None)
    ld, unit = qkv.stride()
    if n_kv != kv or n_heads <= 0 or width != (n_heads + 2 * n_kv) * hd or unit != 1:
        _refuse(what, "qkv must be [tokens, (n_heads + 2 n_kv) * head_dim] with the pages' kv heads and unit column stride")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != hd // 2:
        _refuse(what, "cos and sin must be [positions, head_dim / 2]")
    ld_rope, unit = cos.stride()
    if cos.shape[0] == 1:  # (a single row's stride means nothing)
        ld_rope = 0
    elif sin.stride()[0] != ld_rope:
        _refuse(what, "cos and sin must have the same row stride")
    if unit != 1 or sin.stride()[1] != 1:
        _refuse(what, "cos and sin must have unit column stride")
    if offset < 0:
        _refuse(what, "offset must not be negative")
    dtype = qkv.dtype
    if dtype is not k_pages.dtype and scales is None:
        _wrong_type(what, f"qkv is {dtype}, the pages are {k_pages.dtype}")
    if dtype not in _DTYPES:
        _wrong_type(what, f"qkv must be fp16 or bf16, got {dtype}")
    f32 = cos.dtype is torch.float32
    if sin.dtype is not cos.dtype or not (f32 or cos.dtype is dtype):
        _wrong_type(what, "cos and sin must be fp32 or qkv's type")
    if out is not None and (out.shape != (T, n_heads, hd) or not out.is_contiguous() or out.dtype is not dtype):
        _refuse(what, "out must be a contiguous [tokens, n_heads, head_dim] of qkv's type")
    device = _lib.current_device_of(what, (qkv, k_pages, v_pages, page_table, lengths, starts, cos, sin, out))
    q = qkv.new_empty_strided((T, n_heads, hd), (n_heads * hd, hd, 1)) if out is None else out
    args = (
        qkv.data_ptr(), ld, k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, page_table.data_ptr(),
        ld_table, table_width, lengths.data_ptr(), 0 if starts is None else starts.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        f32, ld_rope, cos.shape[0], offset, q.data_ptr(), T, B, n_heads, n_kv, hd,
        _DTYPES[dtype], _raw_stream(device))
    if scales is None:
        status = _lib.lib().dk_paged_append(_lib.PAGED_APPEND_ARGS.pack(*args))
    else:
        status = _lib.lib().dk_paged_append_fp4(_lib.PAGED_APPEND_FP4_ARGS.pack(*args, *scales))
    if status:
        _lib.check(status, what)
    return q


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(T, B, nq, nkv, hd, dtype, ragged, prefix, device, positions):
    n = ctypes.c_uint64(0)  # (`device`: the current one, whose number of SMs the size depends on)
    if positions:  # a cache of 4-bit codes
        _lib.call("dk_paged_attention_fp4_workspace_bytes", T, B, nq, nkv, hd, dtype, ragged, prefix, positions, ctypes.byref(n))
    else:
        _lib.call("dk_paged_attention_workspace_bytes", T, B, nq, nkv, hd, dtype, ragged, prefix, ctypes.byref(n))
    return int(n.value)


def _attend(what, entry, q, k_pages, v_pages, prefix_table, prefix_len, page_table, lengths, starts, window, sinks, scale, out,
            scales=None):
    """`scales`: (k_scale, v_scale) of a cache of 4-bit codes, or None."""
    if q.dim() != 3:
        _refuse(what, "q must be [tokens, heads, head_dim]")
    T, nq, width = q.shape
    n_pages, n_kv, page, hd, B, ld_table, table_width = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, T,
                                                                     scales is not None)
    ld, by_head, unit = q.stride()
    if width != hd or unit != 1 or by_head != hd and nq > 1 or ld < nq * hd and T > 1:
        _refuse(what, "q must be [tokens, heads, head_dim], a token's heads side by side and tokens apart from each other")
    if nq <= 0 or nq % n_kv or nq // n_kv > MAX_GROUP:
        _refuse(what, f"query heads must be a multiple of the kv heads, at most {MAX_GROUP} for each")
    dtype = q.dtype
    if dtype is not k_pages.dtype and scales is None:
        _wrong_type(what, f"q is {dtype}, the pages are {k_pages.dtype}")
    if dtype not in _DTYPES:
        _wrong_type(what, f"q must be fp16 or bf16, got {dtype}")
    if out is None:
        out = q.new_empty_strided((T, nq, hd), (nq * hd, hd, 1))
    elif out.shape != q.shape or not out.is_contiguous() or out.dtype is not dtype:
        _refuse(what, "out must be a contiguous tensor of q's shape and type")
    prefix_at = 0
    if prefix_len:
        if prefix_len < 0 or prefix_table.dim() != 1 or not prefix_table.is_contiguous() or \
                prefix_table.shape[0] * page < prefix_len:
            _refuse(what, "prefix_table must list the pages of prefix_len positions")
        if prefix_table.dtype is not _INT32:
            _wrong_type(what, "prefix_table must be int32")
        prefix_at = prefix_table.data_ptr()
    device = _lib.current_device_of(what, (q, k_pages, v_pages, page_table, lengths, starts, prefix_table, out))
    code = _DTYPES[dtype]
    # the prefix's length does not change the size, only whether there is one
    nbytes = _workspace_bytes(T, B, nq, n_kv, hd, code, starts is not None, 1 if prefix_len else 0, device,
                              0 if scales is None else table_width * page)
    ws = q.new_empty_strided(((nbytes + 1) // 2,), (1,))  # (of a 16-bit type)
    args = (
        q.data_ptr(), ld, k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, prefix_at, prefix_len,
        page_table.data_ptr(), ld_table, table_width, lengths.data_ptr(),
        0 if starts is None else starts.data_ptr(), window, sinks, hd ** -0.5 if scale is None else scale, out.data_ptr(), T,
        B, nq, n_kv, hd, code, ws.data_ptr(), nbytes, _raw_stream(device))
    pack = _lib.PAGED_ATTENTION_ARGS.pack(*args) if scales is None else _lib.PAGED_ATTENTION_FP4_ARGS.pack(*args, *scales)
    status = getattr(_lib.lib(), entry)(pack)
    if status:
        _lib.check(status, what)
    return out


def paged_attention(q, k_pages, v_pages, page_table, lengths, starts=None, window=0, sinks=0, scale=None, out=None):
    """Attention of q [T, n_heads, head_dim] (tokens any stride apart) over the pages: the row at position p sees the
    positions j <= p of its sequence, with window > 0 only those with j > p - window or j < sinks. Returns [T,
    n_heads, head_dim] contiguous (`out` if given); a row that sees nothing, or belongs to no sequence, is zero. scale: any
    number, head_dim ** -0.5 if None. Pages that no row sees are not read, and their table entries may hold anything; a
    visible position without a page in the pool (read as zeros) or past the table (left out) sets the device error
    DK_DEVERR_BAD_POSITION. With several tokens of a sequence in one call, the keys and values that one of them sees have to
    be finite for the others too."""
    if window < 0 or sinks < 0:
        _refuse("paged_attention", "window and sinks must not be negative")
    return _attend("paged_attention", "dk_paged_attention", q, k_pages, v_pages, None, 0, page_table, lengths, starts, window,
                   sinks, scale, out)


def shared_prefix_attention(q, k_pages, v_pages, prefix_table, prefix_len, page_table, lengths, starts=None, scale=None,
                            out=None):
    """Attention of a batch whose sequences share a prefix: every row of q [T, n_heads, head_dim] sees the prefix's
    prefix_len positions (in the pages prefix_table lists, int32 [>= pages of the prefix]) and, causally, its own
    sequence's positions (page_table, lengths, starts: counted without the prefix); a row of an unused slot or of no
    sequence sees the prefix alone. The prefix's keys and values are read once for all rows. Returns [T, n_heads,
    head_dim] (`out` if given). With starts, all results pass through a workspace in fp32: 1 KB x head_dim for each kv head
    and tile of up to 256 rows, of the prefix's and of the sequences' (1 GB for 32768 tokens of 28 heads over 4)."""
    if prefix_len == 0:
        return paged_attention(q, k_pages, v_pages, page_table, lengths, starts, scale=scale, out=out)
    return _attend("shared_prefix_attention", "dk_shared_prefix_attention", q, k_pages, v_pages, prefix_table, prefix_len,
                   page_table, lengths, starts, 0, 0, scale, out)
