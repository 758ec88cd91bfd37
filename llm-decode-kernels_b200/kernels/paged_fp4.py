"""The serving ops of kernels.paged over a KV cache held in 4 bits: 9/32 of its bytes, so 3.5 times the context in the same memory
and about as much more of it read per second.

A value of the cache is code * scale * k_scale (v_scale for v): a 4-bit E2M1 code (a sign and 0, 0.5, 1, 1.5, 2, 3, 4 or 6), an E4M3
scale for each 16 dims of a position, and one power of two for a whole pool, 1 unless given, which puts values of another size
in the scales' range (2^-9 to 448: largest magnitudes in 16 dims from 0.01 to 2688 times the power). code * scale is exact in fp16 and
bf16, and attention computes with just these numbers; only appending rounds.

A pool is uint8 [n_pages, n_kv, page_size, 9/16 head_dim] (`fp4_pages`). The block of a (page, kv head) holds first the codes,
head_dim / 2 bytes a position with dim 2 i in the low half of byte i, then the scales, head_dim / 16 bytes a position. Page
tables, lengths, starts, their types, and what unused slots and rows of no sequence do are those of kernels.paged; q, qkv and
results are fp16 or bf16. The reference's cache is fp16 (kernels/e2e/model.py:192); it has no counterpart of these ops.
"""

from __future__ import annotations

import functools
import math

import torch

from kernels import _lib
from kernels.paged import _DTYPES, _append, _attend, _cache_shape, _raw_stream, _refuse, _wrong_type


def fp4_pages(n_pages: int, n_kv: int, page_size: int, head_dim: int, device=None) -> torch.Tensor:
    """A pool of 4-bit pages, uninitialized like torch.empty: positions count once they are appended."""
    if head_dim not in (64, 128):
        raise ValueError("fp4_pages: head_dim must be 64 or 128")
    return torch.empty(n_pages, n_kv, page_size, head_dim * 9 // 16, dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)  # (of numbers only: a model has a pair of them)
def _powers(what, k_scale: float, v_scale: float):
    for x in (k_scale, v_scale):
        if not (isinstance(x, (int, float)) and 2.0 ** -64 <= x <= 2.0 ** 64 and math.frexp(x)[0] == 0.5):
            _refuse(what, "k_scale and v_scale must be numbers, powers of two from 2^-64 to 2^64")
    return float(k_scale), float(v_scale)


def paged_append_fp4(qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts=None, offset=0, k_scale=1.0,
                     v_scale=1.0, out=None):
    """`paged_append` into a 4-bit cache: rotates q and k of qkv [T, (n_heads + 2 n_kv) * head_dim] and writes k and v. Each 16 dims of
    a position get scale = E4M3(max |x| / 6) and codes E2M1(x / scale) of x / k_scale (x / v_scale for v), rounded to nearest,
    ties to even; what is too large saturates, a NaN makes its 16 dims NaN. The rotation of k is computed in fp64, where its
    products are exact, rounded to fp32 and from there to qkv's type, so that the codes do not hang on the order of operations. Returns the rotated q [T, n_heads, head_dim] (`out`)."""
    what = "paged_append_fp4"
    return _append(what, qkv, k_pages, v_pages, page_table, lengths, cos, sin, n_heads, n_kv, starts, offset, out,
                   _powers(what, k_scale, v_scale))


def paged_read_fp4(k_pages, v_pages, page_table, lengths, starts=None, tokens=None, dtype=torch.float16, k_scale=1.0, v_scale=1.0,
                   out=None):
    """Read positions back: k and v [T, n_kv, head_dim] of `dtype` (`out`: a pair of such tensors). The rows are the tokens of a call
    with these lengths and starts: without starts each sequence's last position (T = B); with them `tokens` rows, of which
    starts[b]..starts[b+1] are the last ones of sequence b (its length of them: the whole sequence). Values are exact unless
    k_scale or v_scale takes them out of dtype's range. Rows of no sequence, or before a sequence's first position, are zero; a
    position without a page in the pool is zero and sets the device error DK_DEVERR_BAD_POSITION."""
    what = "paged_read_fp4"
    if out is not None:
        if len(out) != 2:
            _refuse(what, "out must be two contiguous [tokens, n_kv, head_dim] of one type")
        rows, dtype = out[0].shape[0], out[0].dtype
        if tokens is not None and tokens != rows:
            _refuse(what, f"out has {rows} rows, tokens says {tokens}")
        tokens = rows
    elif tokens is None:
        if starts is not None:
            _refuse(what, "with starts, tokens says how many rows there are")
        tokens = page_table.shape[0]
    if tokens < 0:
        _refuse(what, "tokens must not be negative")
    n_pages, n_kv, page, hd, B, ld_table, table_width = _cache_shape(what, k_pages, v_pages, page_table, lengths, starts, tokens, True)
    k_scale, v_scale = _powers(what, k_scale, v_scale)
    if dtype not in _DTYPES:
        _wrong_type(what, f"values are fp16 or bf16, not {dtype}")
    shape = (tokens, n_kv, hd)
    if out is not None and not all(x.shape == shape and x.is_contiguous() and x.dtype is dtype for x in out):
        _refuse(what, "out must be two contiguous [tokens, n_kv, head_dim] of one type")
    device = _lib.current_device_of(what, (k_pages, v_pages, page_table, lengths, starts, *(out or ())))
    if out is None:
        k = k_pages.new_empty_strided(shape, (n_kv * hd, hd, 1), dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = out
    status = _lib.lib().dk_paged_read_fp4(_lib.PAGED_READ_FP4_ARGS.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page, page_table.data_ptr(), ld_table, table_width,
        lengths.data_ptr(), 0 if starts is None else starts.data_ptr(), k_scale, v_scale, k.data_ptr(), v.data_ptr(), tokens, B,
        n_kv, hd, _DTYPES[dtype], _raw_stream(device)))
    if status:
        _lib.check(status, what)
    return k, v


def paged_attention_fp4(q, k_pages, v_pages, page_table, lengths, starts=None, window=0, sinks=0, scale=None, k_scale=1.0,
                        v_scale=1.0, out=None):
    """`paged_attention` over a 4-bit cache: q [T, n_heads, head_dim] -> [T, n_heads, head_dim] of q's type (`out`), with its masks,
    its device error for visible positions without a page, and its rows that see nothing."""
    what = "paged_attention_fp4"
    if window < 0 or sinks < 0:
        _refuse(what, "window and sinks must not be negative")
    return _attend(what, "dk_paged_attention_fp4", q, k_pages, v_pages, None, 0, page_table, lengths, starts, window, sinks, scale,
                   out, _powers(what, k_scale, v_scale))


def shared_prefix_attention_fp4(q, k_pages, v_pages, prefix_table, prefix_len, page_table, lengths, starts=None, scale=None,
                                k_scale=1.0, v_scale=1.0, out=None):
    """`shared_prefix_attention` over a 4-bit cache (the prefix's pages and the sequences' own lie in the same two pools)."""
    if prefix_len == 0:
        return paged_attention_fp4(q, k_pages, v_pages, page_table, lengths, starts, scale=scale, k_scale=k_scale, v_scale=v_scale,
                                   out=out)
    what = "shared_prefix_attention_fp4"
    return _attend(what, "dk_shared_prefix_attention_fp4", q, k_pages, v_pages, prefix_table, prefix_len, page_table, lengths, starts,
                   0, 0, scale, out, _powers(what, k_scale, v_scale))
