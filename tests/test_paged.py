"""The paged-cache ops (kernels.paged, C-ABI dk_paged_append, dk_paged_attention, dk_shared_prefix_attention) against
plain 64-bit implementations, at the sizes and masks where they can go wrong, and their refusals."""

import math

import pytest
import torch

from _paged import UNIT, Case, assert_within

F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------------------------------------ append
def _rope(positions, hd, dtype=torch.float32):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,table_type,offset", [
    ([(1, 1)], 12, 2, 128, 16, F16, torch.float32, 0),
    ([(1, 17), (1, 300), (1, 64), (1, 65)], 28, 4, 128, 64, BF16, torch.float32, 0),
    ([(5, 5), (0, 9), (33, 70), (1, 1), (100, 129)], 7, 1, 64, 32, F16, F16, 0),
    ([(3, 250), (129, 400)], 8, 8, 64, 256, BF16, BF16, 11),
    ([(1, 0), (1, 40), (1, -3)], 4, 1, 128, 128, F16, torch.float32, 1000),  # unused slots of the batch
])
def test_append(sizes, nq, nkv, hd, page, dtype, table_type, offset):
    from kernels import _lib
    from kernels.paged import paged_append

    c = Case(sizes, nq, nkv, hd, page, dtype, spoil=False)
    qkv = torch.randn(c.T, (nq + 2 * nkv) * hd + 8, device="cuda").to(dtype)[:, :-8]  # strided rows
    cos, sin = _rope(max(n for _, n in sizes) + offset + 1, hd, table_type)
    k, v = c.k.clone(), c.v.clone()
    _lib.clear_device_error()
    q = paged_append(qkv, k, v, c.table, c.lengths, cos, sin, nq, nkv, starts=c.starts, offset=offset)
    assert _lib.device_error() == 0
    x = qkv.double().cpu().view(c.T, nq + 2 * nkv, hd)
    want_k, want_v, u = c.k.double().cpu(), c.v.double().cpu(), UNIT[dtype]
    slack_k = torch.zeros_like(want_k)
    t = 0
    for b, (new, n) in enumerate(sizes):
        for i in range(new):
            p = n - new + i
            if p < 0:
                assert not q[t].any()
                t += 1
                continue
            a, s = cos[p + offset].double().cpu(), sin[p + offset].double().cpu()
            lo, hi = x[t, :nq + nkv, :hd // 2], x[t, :nq + nkv, hd // 2:]
            turned = torch.cat([lo * a - hi * s, hi * a + lo * s], -1)
            # fp32: two products and a sum, each rounded; then once to the type
            size = torch.cat([(lo * a).abs() + (hi * s).abs(), (hi * a).abs() + (lo * s).abs()], -1)
            slack = u * turned.abs() + (2.0 ** -23 + 2.0 ** -24 * u) * size + 2.0 ** -25
            assert ((q[t].double().cpu() - turned[:nq]).abs() <= slack[:nq]).all()
            row = c.table[b, p // page].long().item()
            want_k[row, :, p % page], slack_k[row, :, p % page] = turned[nq:], slack[nq:]
            want_v[row, :, p % page] = x[t, nq + nkv:]
            t += 1
    assert ((k.double().cpu() - want_k).abs() <= slack_k).all()  # nothing else in the pool changed
    assert torch.equal(v.double().cpu(), want_v)


@pytest.mark.gpu
def test_append_without_a_page_or_an_angle_writes_nothing():
    from kernels import _lib
    from kernels.paged import paged_append

    c = Case([(1, 20), (1, 5)], spoil=False)
    cos, sin = _rope(64, 128)
    qkv = torch.randn(2, 16 * 128, device="cuda").half()
    for spoil in ("table", "pool", "angle"):
        k, v, table = c.k.clone(), c.v.clone(), c.table.clone()
        table[:, :] = {"table": -1, "pool": c.k.shape[0], "angle": 0}[spoil]
        rows = slice(0, 3) if spoil == "angle" else slice(0, 64)
        _lib.clear_device_error()
        paged_append(qkv, k, v, table, c.lengths, cos[rows], sin[rows], 12, 2)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        assert torch.equal(k, c.k) and torch.equal(v, c.v)


# ------------------------------------------------------------------------------------------ attention
DECODE = [
    # sizes, nq, nkv, hd, page, dtype, window, sinks
    ([(1, 1)], 12, 2, 128, 16, F16, 0, 0),
    ([(1, 640)], 12, 2, 128, 16, F16, 0, 0),
    ([(1, 63), (1, 64), (1, 65), (1, 1), (1, 0), (1, 129)], 28, 4, 128, 64, BF16, 0, 0),
    ([(1, 1000), (1, 3), (1, 517)], 16, 1, 128, 32, F16, 0, 0),
    ([(1, 700), (1, 31)], 8, 8, 64, 128, BF16, 0, 0),
    ([(1, 300)] * 70, 4, 1, 64, 16, F16, 0, 0),
    ([(1, 777), (1, 40), (1, 5)], 12, 2, 128, 16, F16, 100, 4),
    ([(1, 777), (1, 40), (1, 128)], 14, 2, 128, 64, BF16, 1, 0),
    ([(1, 777), (1, 100)], 7, 1, 128, 32, F16, 64, 70),  # the sinks reach into the second chunk
    ([(1, 90), (1, 300)], 4, 2, 64, 16, F16, 1 << 30, 3),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,window,sinks", DECODE)
def test_attention_one_token(sizes, nq, nkv, hd, page, dtype, window, sinks):
    from kernels import _lib
    from kernels.paged import paged_attention

    c = Case(sizes, nq, nkv, hd, page, dtype, seed=1)
    _lib.clear_device_error()
    out = paged_attention(c.q, c.k, c.v, c.table, c.lengths, window=window, sinks=sinks)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, paged_attention(c.q, c.k, c.v, c.table, c.lengths, window=window, sinks=sinks))


RAGGED = [
    ([(1, 1), (2, 2)], 12, 2, 128, 16, F16, 0, 0),
    ([(7, 7), (0, 30), (130, 200), (1, 90), (64, 64)], 12, 2, 128, 16, BF16, 0, 0),
    ([(300, 300)], 28, 4, 128, 64, F16, 0, 0),
    ([(200, 430), (33, 33)], 16, 1, 128, 32, BF16, 0, 0),
    ([(150, 280), (129, 129)], 8, 8, 64, 128, F16, 0, 0),
    ([(257, 300), (20, 400)], 5, 1, 64, 256, BF16, 0, 0),
    ([(5, 3), (4, 0), (6, 6)], 12, 2, 128, 16, F16, 0, 0),  # fewer positions than tokens: rows that see nothing
    ([(260, 400), (50, 300), (3, 3)], 12, 2, 128, 16, F16, 37, 4),
    ([(300, 300)], 14, 2, 128, 64, BF16, 1, 2),
    ([(140, 500)], 7, 1, 64, 32, F16, 128, 0),
    ([(140, 700)], 3, 1, 128, 32, F16, 130, 129),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,window,sinks", RAGGED)
def test_attention_ragged(sizes, nq, nkv, hd, page, dtype, window, sinks):
    from kernels import _lib
    from kernels.paged import paged_attention

    c = Case(sizes, nq, nkv, hd, page, dtype, seed=2, one_token=False)
    _lib.clear_device_error()
    out = paged_attention(c.q, c.k, c.v, c.table, c.lengths, starts=c.starts, window=window, sinks=sinks)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, paged_attention(c.q, c.k, c.v, c.table, c.lengths, starts=c.starts, window=window, sinks=sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq", [(128, 8), (64, 8), (128, 80)])
def test_attention_long_rings(hd, nq):
    """Many more chunks per CTA than its ring has slots, call after call without a host wait in between: every call gives
    the first one's bits, and no bounded wait gives up."""
    from kernels import _lib
    from kernels.paged import paged_attention

    sizes = [(1, 4000 + 97 * b) for b in range(10)]
    c = Case(sizes, nq=nq, nkv=8, hd=hd, page=64, seed=8, spoil=False)
    _lib.clear_device_error()
    first = paged_attention(c.q, c.k, c.v, c.table, c.lengths)
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(200):
        same &= (paged_attention(c.q, c.k, c.v, c.table, c.lengths) == first).all()
    assert same.item() and _lib.device_error() == 0
    few = Case(sizes[:2], nq=nq, nkv=8, hd=hd, page=64, seed=9)
    assert_within(paged_attention(few.q, few.k, few.v, few.table, few.lengths), *few.attention())


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
def test_attention_leaves_freed_pages_alone(one_token):
    """Pages outside the window and the sinks may be freed: their table entries point nowhere."""
    from kernels.paged import paged_attention

    sizes = [(1, 700), (1, 130)] if one_token else [(9, 700), (40, 130)]
    c = Case(sizes, seed=3, one_token=one_token)
    window, sinks = 50, 4
    want = c.attention(window, sinks)
    for b, (new, n) in enumerate(sizes):
        first, last = 1, (n - new + 1 - window) // c.page
        for i in range(first, last):
            page = c.table[b, i].long().item()
            c.k[page], c.v[page] = math.nan, math.nan
        c.table[b, first:last] = torch.tensor([-1, 1 << 30]).repeat(last)[:last - first].int()
    out = paged_attention(c.q, c.k, c.v, c.table, c.lengths, starts=c.starts, window=window, sinks=sinks)
    assert_within(out, *want)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,window,sinks", [([(1, 400), (1, 31)], 0, 0), ([(70, 200), (3, 90)], 40, 2)])
def test_attention_strides_scale_stream_and_graph(sizes, window, sinks):
    """q rows inside a wider tensor, a table with spare columns, another scale, a side stream, a captured call."""
    from kernels.paged import paged_attention

    c = Case(sizes, seed=4)
    wide = torch.zeros(c.T, c.nq + 5, c.hd, dtype=c.dtype, device="cuda")
    wide[:, :c.nq] = c.q
    table = torch.full((len(sizes), c.table.shape[1] + 40), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    args = (wide[:, :c.nq], c.k, c.v, table[:, :c.table.shape[1] + 3], c.lengths)
    more = dict(starts=c.starts, window=window, sinks=sinks, scale=0.2)
    want = c.attention(window, sinks, scale=0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged_attention(*args, **more)
    torch.cuda.current_stream().wait_stream(side)
    assert_within(out, *want)
    graph, kept = torch.cuda.CUDAGraph(), torch.empty_like(out)
    with torch.cuda.graph(graph):
        paged_attention(*args, out=kept, **more)
    graph.replay()
    assert torch.equal(kept, out)


@pytest.mark.gpu
def test_attention_long_context_and_masked_extremes():
    """The type's lowest value and infinities in k or v at masked positions; scores far apart; long contexts."""
    from kernels.paged import paged_attention

    c = Case([(1, 5000), (1, 2)], nq=6, nkv=1, page=128, seed=5)
    c.q[0] *= 3
    out = paged_attention(c.q, c.k, c.v, c.table, c.lengths)
    assert_within(out, *c.attention())
    low = Case([(1, 100)], nq=6, nkv=1, seed=6, spoil=False)
    want = low.attention(16, 2)
    page = low.table[0].long()
    for j in range(2, 84):  # neither a sink nor in the window
        low.k[page[j // 16], :, j % 16] = torch.finfo(F16).min
        low.v[page[j // 16], :, j % 16] = math.inf
    assert_within(paged_attention(low.q, low.k, low.v, low.table, low.lengths, window=16, sinks=2), *want)


# ------------------------------------------------------------------------------------------ shared prefix
@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[(1, 300)], [(1, 300), (1, 0), (1, 31)], [(9, 5), (4, 200), (3, 0)]])
def test_attention_windows_past_every_position(sizes):
    """A window as long as the table or longer masks nothing, up to the largest; rows before the first position are empty."""
    from kernels.paged import paged_attention

    c = Case(sizes, one_token=all(n == 1 for n, _ in sizes))
    args = (c.q, c.k, c.v, c.table, c.lengths, c.starts)
    plain = paged_attention(*args)
    exact, tol = c.attention()
    assert_within(plain, exact, tol)
    for window in (c.table.shape[1] * c.page, 2 ** 31 - 1):
        for sinks in (0, 4, 2 ** 31 - 1):
            assert torch.equal(paged_attention(*args, window=window, sinks=sinks), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("sizes", [[(1, 700), (1, 101), (1, 100), (1, 3)], [(60, 700), (50, 120), (2, 100), (9, 9)]])
def test_attention_sinks_beside_the_window(page, sizes):
    """Sinks that end in their page, at its end, just before the window's first page, in it and beyond: the positions between
    are skipped, not seen."""
    from kernels.paged import paged_attention

    c = Case(sizes, nq=4, nkv=2, hd=64, page=page)
    for sinks in (0, 1, 16, 17, 64, 256, 511, 512, 513, 599, 600, 690):
        exact, tol = c.attention(window=100, sinks=sinks)
        assert_within(paged_attention(c.q, c.k, c.v, c.table, c.lengths, c.starts, window=100, sinks=sinks), exact, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(torch.float16, 64), (torch.bfloat16, 128)])
@pytest.mark.parametrize("sizes,prefix", [([(1, 9000)], 0), ([(5, 9000)], 0), ([(3, 5000), (70, 6000), (1, 40)], 0),
                                          ([(1, 3), (1, 700)], 9000), ([(4, 9), (30, 2000)], 5001)])
def test_units_cut_into_many_pieces(sizes, prefix, dtype, hd):
    """Few rows over long caches: every CTA works on the same units, whose many partial results are joined in parts."""
    from kernels.paged import paged_attention, shared_prefix_attention

    c = Case(sizes, nq=6, nkv=2, hd=hd, page=32, dtype=dtype, prefix=prefix)
    exact, tol = c.attention()
    if prefix:
        got = shared_prefix_attention(c.q, c.k, c.v, c.prefix_table, prefix, c.table, c.lengths, c.starts)
    else:
        got = paged_attention(c.q, c.k, c.v, c.table, c.lengths, c.starts)
    assert_within(got, exact, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_one_token_of_any_stride(ragged):
    """The row stride of a single token means nothing, whatever it is."""
    from kernels.paged import paged_append, paged_attention

    c = Case([(1, 77)], one_token=not ragged)
    odd = c.q.as_strided(c.q.shape, (3, c.hd, 1))
    exact, tol = c.attention()
    assert_within(paged_attention(odd, c.k, c.v, c.table, c.lengths, c.starts), exact, tol)
    qkv = torch.randn(1, (c.nq + 2 * c.nkv) * c.hd, device="cuda", dtype=c.dtype)
    angle = torch.rand(100, c.hd // 2, device="cuda")
    a = paged_append(qkv, c.k.clone(), c.v.clone(), c.table, c.lengths, angle.cos(), angle.sin(), c.nq, c.nkv, c.starts)
    b = paged_append(qkv.as_strided(qkv.shape, (5, 1)), c.k, c.v, c.table, c.lengths, angle.cos(), angle.sin(), c.nq, c.nkv,
                     c.starts)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,prefix,nq,nkv,hd,page,dtype", [
    ([(1, 1)], 1, 12, 2, 128, 16, F16),
    ([(1, 40), (1, 1), (1, 65)], 525, 12, 2, 128, 16, F16),
    ([(1, 3)] * 50, 200, 28, 4, 128, 64, BF16),
    ([(1, 20), (1, 0), (1, 7)], 64, 8, 8, 64, 32, F16),  # an unused slot: the prefix alone
    ([(2, 30), (5, 5), (1, 90)], 333, 16, 1, 128, 32, BF16),
    ([(40, 70), (100, 100)], 130, 7, 1, 64, 128, F16),
    ([(1, 5)] * 9, 2500, 5, 1, 128, 256, F16),
])
def test_shared_prefix(sizes, prefix, nq, nkv, hd, page, dtype):
    from kernels import _lib
    from kernels.paged import paged_attention, shared_prefix_attention

    c = Case(sizes, nq, nkv, hd, page, dtype, seed=7, prefix=prefix)
    _lib.clear_device_error()
    out = shared_prefix_attention(c.q, c.k, c.v, c.prefix_table, prefix, c.table, c.lengths, starts=c.starts)
    assert _lib.device_error() == 0
    exact, tol = c.attention()
    assert_within(out, exact, tol)
    again = shared_prefix_attention(c.q, c.k, c.v, c.prefix_table, prefix, c.table, c.lengths, starts=c.starts)
    assert torch.equal(out, again)
    none = shared_prefix_attention(c.q, c.k, c.v, c.prefix_table, 0, c.table, c.lengths, starts=c.starts)
    assert torch.equal(none, paged_attention(c.q, c.k, c.v, c.table, c.lengths, starts=c.starts))


# ------------------------------------------------------------------------------------------ refusals
def _cpu_case(**more):
    return Case([(1, 20), (1, 5)], spoil=False, device="cpu", **more)


def test_refusals_without_a_gpu():
    """Extents, types and layouts the kernels cannot take are refused before any device work."""
    from kernels.paged import paged_append, paged_attention, shared_prefix_attention

    c = _cpu_case()
    args = [c.q, c.k, c.v, c.table, c.lengths]
    starts = torch.tensor([0, 1, 2], dtype=torch.int32)

    def attend(error, *at, **more):
        a = list(args)
        for i, x in at:
            a[i] = x
        with pytest.raises(error):
            paged_attention(*a, **more)

    attend(RuntimeError)  # on the CPU
    attend(ValueError, (0, c.q[:1]))  # a token per sequence
    attend(ValueError, (0, c.q[..., :64]))
    attend(ValueError, (0, c.q[:, :5]))  # 5 query heads over 2 kv heads
    attend(ValueError, (0, torch.zeros(2, 34, 128).half()))  # 17 query heads for each kv head
    attend(ValueError, (0, c.q.transpose(1, 2).contiguous().transpose(1, 2)))
    attend(ValueError, (0, c.q[:1].expand(2, -1, -1)))  # overlapping tokens
    attend(ValueError, (1, c.k[:, :, :8].contiguous()), (2, c.v[:, :, :8].contiguous()))
    attend(ValueError, (1, c.k[:-1]))
    attend(ValueError, (1, c.k.transpose(0, 1)), (2, c.v.transpose(0, 1)))
    attend(ValueError, (1, c.k[..., :32].contiguous()), (2, c.v[..., :32].contiguous()))
    attend(ValueError, (3, c.table[:1]))
    attend(ValueError, (4, c.lengths[:1]))
    attend(ValueError, starts=starts[:2])
    attend(ValueError, window=-1)
    attend(ValueError, sinks=-1)
    attend(ValueError, out=torch.zeros(2, 12, 64).half())
    attend(RuntimeError, (0, c.q.float()))
    attend(RuntimeError, (1, c.k.float()), (2, c.v.float()))
    attend(RuntimeError, (3, c.table.long()))
    attend(RuntimeError, starts=starts.long())
    with pytest.raises(ValueError):
        shared_prefix_attention(c.q, c.k, c.v, c.table[0], 1000, c.table, c.lengths)
    with pytest.raises(ValueError):
        shared_prefix_attention(c.q, c.k, c.v, c.table[0], -1, c.table, c.lengths)
    with pytest.raises(RuntimeError):
        shared_prefix_attention(c.q, c.k, c.v, c.table[0].long(), 10, c.table, c.lengths)

    qkv, cos = torch.zeros(2, 16 * 128).half(), torch.zeros(40, 64)
    good = dict(qkv=qkv, cos=cos, sin=cos, n_heads=12, n_kv=2)

    def append(error, **more):
        a = {**good, **more}
        with pytest.raises(error):
            paged_append(a["qkv"], c.k, c.v, c.table, c.lengths, a["cos"], a["sin"], a["n_heads"], a["n_kv"],
                         offset=a.get("offset", 0), out=a.get("out"))

    append(RuntimeError)  # on the CPU
    append(ValueError, qkv=qkv[:, :-128])
    append(ValueError, qkv=qkv[:1])
    append(ValueError, n_kv=4)
    append(ValueError, cos=torch.zeros(40, 128), sin=torch.zeros(40, 128))
    append(ValueError, sin=torch.zeros(39, 64))
    append(ValueError, offset=-1)
    append(ValueError, out=torch.zeros(2, 12, 64).half())
    append(RuntimeError, qkv=qkv.bfloat16())
    append(RuntimeError, cos=cos.bfloat16(), sin=cos.bfloat16())


def test_c_entries_refuse_without_a_gpu():
    """The C entry points return a status and a message for what they cannot take, before any CUDA call."""
    import ctypes

    from kernels import _lib

    h, n = _lib.lib(), ctypes.c_uint64(0)

    def attend(**more):
        a = dict(T=2, B=2, nq=12, nkv=2, hd=128, page=16, dtype=0, ldq=1536, pages=4, width=2)
        a.update(more)
        return h.dk_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(
            0, a["ldq"], 0, 0, a["pages"], a["page"], 0, 0, 0, a["width"], a["width"], 0, 0, 0, 0, 1.0, 0, a["T"], a["B"],
            a["nq"], a["nkv"], a["hd"], a["dtype"], 0, 0, 0))

    def append(page):
        return h.dk_paged_append(_lib.PAGED_APPEND_ARGS.pack(0, 0, 0, 0, 4, page, 0, 2, 2, 0, 0, 0, 0, 1, 64, 10, 0, 0, 3, 2,
                                                             12, 2, 128, 0, 0))

    assert h.dk_paged_attention(None) == -1 and h.dk_shared_prefix_attention(None) == -1 and h.dk_paged_append(None) == -1
    assert attend() == -1 and b"NULL" in h.dk_last_error()
    assert attend(T=3) == -1 and b"one token" in h.dk_last_error()
    assert attend(hd=96) == -3 and b"head_dim" in h.dk_last_error()
    assert attend(page=24) == -3 and b"page_size" in h.dk_last_error()
    assert attend(nq=13) == -3 and attend(nq=34) == -3
    assert attend(dtype=2) == -3
    assert attend(B=5000, T=5000) == -3 and b"sequences" in h.dk_last_error()
    assert attend(ldq=8) == -1 and b"overlap" in h.dk_last_error()
    assert attend(pages=1 << 26) == -1 and b"2^31" in h.dk_last_error()
    assert attend(width=1 << 27) == -1
    assert h.dk_paged_attention_workspace_bytes(2, 2, 12, 2, 96, 0, 0, 0, ctypes.byref(n)) == -3
    assert append(16) == -1 and b"one token" in h.dk_last_error()
    assert append(20) == -3 and b"page_size" in h.dk_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 128), (BF16, 64)])
@pytest.mark.parametrize("scale", [0.0, -0.15, 1e-60])
@pytest.mark.parametrize("sizes,prefix,window,sinks", [
    ([(1, 200), (1, 3)], 0, 0, 0), ([(60, 300), (9, 9), (4, 2)], 0, 0, 0), ([(140, 400), (1, 90)], 0, 50, 3),
    ([(1, 70), (1, 0)], 200, 0, 0), ([(5, 30), (50, 60)], 333, 0, 0),
])
def test_scale_of_any_sign(sizes, prefix, window, sinks, scale, dtype, hd):
    """A scale of zero weighs the visible positions alike, a negative one the smallest products most (1e-60 is zero in fp32);
    masked positions stay out of it. One token each, ragged rows and a shared prefix run different kernels."""
    from kernels.paged import paged_attention, shared_prefix_attention

    c = Case(sizes, nq=6, nkv=2, hd=hd, page=32, dtype=dtype, prefix=prefix, seed=10)
    exact, tol = c.attention(window, sinks, scale=scale)
    if prefix:
        got = shared_prefix_attention(c.q, c.k, c.v, c.prefix_table, prefix, c.table, c.lengths, c.starts, scale=scale)
    else:
        got = paged_attention(c.q, c.k, c.v, c.table, c.lengths, c.starts, window=window, sinks=sinks, scale=scale)
    assert_within(got, exact, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("before,after", [(0, 4), (2, 0), (1, 3)])
def test_append_rows_outside_starts(before, after):
    """Rows before starts[0] and from starts[B] on (a captured call of more rows than the step has) belong to no sequence: they
    append nothing and their q is zero, whatever the last slot's table row lists."""
    from kernels import _lib
    from kernels.paged import paged_append

    sizes = [(3, 20), (2, 40), (1, 0)]
    c = Case(sizes, nkv=2, spoil=False)
    c.table[2] = c.table[0]  # an unused slot with another sequence's pages still in its row
    c.table[:, 2:] = c.table[1, 0]
    cos, sin = _rope(200, 128)
    qkv = torch.randn(before + c.T + after, 16 * 128, device="cuda").half()
    want_k, want_v = c.k.clone(), c.v.clone()
    want = paged_append(qkv[before:before + c.T].contiguous(), want_k, want_v, c.table, c.lengths, cos, sin, 12, 2, starts=c.starts)
    _lib.clear_device_error()
    q = paged_append(qkv, c.k, c.v, c.table, c.lengths, cos, sin, 12, 2, starts=c.starts + before)
    assert _lib.device_error() == 0
    assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v)
    assert torch.equal(q[before:before + c.T], want)
    assert not q[:before].any() and not q[before + c.T:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("before,after,hd", [(0, 700, 128), (2, 0, 64), (3, 5, 128)])
def test_attention_rows_outside_starts(before, after, hd):
    """Rows before starts[0] and from starts[B] on belong to no sequence: zero from attention over the pages, the prefix alone
    from attention with a prefix."""
    from kernels.paged import paged_attention, shared_prefix_attention

    c = Case([(3, 20), (150, 200), (1, 0)], hd=hd, one_token=False, prefix=40)
    q = torch.cat([torch.randn(before, c.nq, hd), torch.zeros(c.T, c.nq, hd), torch.randn(after, c.nq, hd)]).to(c.dtype).cuda()
    q[before:before + c.T] = c.q
    live = slice(before, before + c.T)
    outside = torch.ones(len(q), dtype=torch.bool)
    outside[live] = False
    out = torch.full_like(q, math.nan)
    paged_attention(q, c.k, c.v, c.table, c.lengths, c.starts + before, out=out)
    assert torch.equal(out[live], paged_attention(c.q, c.k, c.v, c.table, c.lengths, c.starts))
    assert not out[outside.cuda()].any()
    out = torch.full_like(q, math.nan)
    shared_prefix_attention(q, c.k, c.v, c.prefix_table, 40, c.table, c.lengths, c.starts + before, out=out)
    alone = Case([(1, 0)] * int(outside.sum()), hd=hd, prefix=40)
    alone.q, alone.k, alone.v, alone.prefix_table = q[outside.cuda()], c.k, c.v, c.prefix_table
    assert_within(out[outside.cuda()], *alone.attention())


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
@pytest.mark.parametrize("window", [0, 30])
def test_attention_reports_positions_without_a_page(one_token, window):
    """A visible position whose table entry names no page of the pool, and a length past the table, set the device error; an
    entry that no row sees does not."""
    from kernels import _lib
    from kernels.paged import paged_attention, shared_prefix_attention

    c = Case([(1, 200), (1, 50)] if one_token else [(40, 200), (3, 50)], one_token=one_token, spoil=False, prefix=100, wide=0)
    page = c.page

    def error(table=None, lengths=None, prefix_table=None):
        table, lengths = c.table if table is None else table, c.lengths if lengths is None else lengths
        _lib.clear_device_error()
        paged_attention(c.q, c.k, c.v, table, lengths, c.starts, window=window, sinks=2)
        code = _lib.device_error()
        if window == 0:
            _lib.clear_device_error()
            shared_prefix_attention(c.q, c.k, c.v, c.prefix_table if prefix_table is None else prefix_table, 100, table, lengths,
                                    c.starts)
            assert _lib.device_error() == (code if prefix_table is None else 3)
        _lib.clear_device_error()
        return code

    assert error() == 0
    for entry in (-1, c.k.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 190 // page] = entry
        assert error(table) == 3  # DK_DEVERR_BAD_POSITION
        table = c.table.clone()
        table[1, 50 // page + 1:] = entry  # after the second sequence's last position
        assert error(table) == 0
        if window == 0:
            wrong = c.prefix_table.clone()
            wrong[2] = entry
            error(prefix_table=wrong)
    assert error(lengths=c.lengths + torch.tensor([table.shape[1] * page - 200 + 1, 0], dtype=torch.int32, device="cuda")) == 3


def test_refuses_a_device_that_is_not_the_current_one(monkeypatch):
    """The library launches on the current device: tensors of another one are refused, by every op, before the C entry."""
    from kernels import _lib, logprobs, paged

    class On:
        def __init__(self, index):
            self.device, self.get_device = f"cuda:{index}", lambda: index

    monkeypatch.setattr(_lib, "_current_device", lambda: 1)
    assert _lib.current_device_of("op", (On(1), None, On(1))) == 1
    for tensors in ((On(0),), (On(0), On(0)), (On(1), On(0)), (On(-1),), (On(2), None)):
        with pytest.raises(RuntimeError, match="op: "):
            _lib.current_device_of("op", tensors)

    def no_entry():
        raise AssertionError("the C entry was reached")

    monkeypatch.setattr(_lib, "lib", no_entry)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    c = _cpu_case()
    cos = torch.zeros(40, 64)
    for call in (lambda: paged.paged_attention(c.q, c.k, c.v, c.table, c.lengths),
                 lambda: paged.shared_prefix_attention(c.q, c.k, c.v, c.table[0], 10, c.table, c.lengths),
                 lambda: paged.paged_append(torch.zeros(2, 16 * 128).half(), c.k, c.v, c.table, c.lengths, cos, cos, 12, 2),
                 lambda: logprobs.token_logprobs(torch.zeros(2, 50), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="current device is cuda:1"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("window", [0, 20])
def test_unused_slots_of_any_negative_length(ragged, window):
    """A length of the type's lowest value is an unused slot like any other <= 0."""
    from kernels import _lib
    from kernels.paged import paged_append, paged_attention

    c = Case([(3, 40), (3, 0), (2, 20), (3, 0)] if ragged else [(1, 40), (1, 0), (1, 20), (1, 0)], one_token=not ragged, spoil=False)
    low = torch.tensor([40, -2 ** 31, 20, -2 ** 31 + 2], dtype=torch.int32, device="cuda")
    want = paged_attention(c.q, c.k, c.v, c.table, c.lengths, c.starts, window=window, sinks=2)
    _lib.clear_device_error()
    assert torch.equal(paged_attention(c.q, c.k, c.v, c.table, low, c.starts, window=window, sinks=2), want)
    cos, sin = _rope(64, 128)
    qkv = torch.randn(c.T, 16 * 128, device="cuda").half()
    k, v = c.k.clone(), c.v.clone()
    want = paged_append(qkv, k, v, c.table, c.lengths, cos, sin, 12, 2, starts=c.starts)
    assert torch.equal(paged_append(qkv, c.k, c.v, c.table, low, cos, sin, 12, 2, starts=c.starts), want)
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    assert _lib.device_error() == 0


def test_tables_whose_positions_pass_31_bits_are_refused():
    """Positions rounded up to whole chunks, and windows before the first position, have to fit 32 bits; products of sizes that
    pass 64 bits do not slip through."""
    from kernels import _lib

    h = _lib.lib()

    def attend(T=2, width=2, page=16, pages=4, window=0, sinks=0):
        return h.dk_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(
            0, 1536, 0, 0, pages, page, 0, 0, 0, width, width, 0, 256, window, sinks, 1.0, 0, T, 2, 12, 2, 128, 0, 0, 0, 0))

    most = (1 << 31) - 1024
    for page in (16, 256):
        assert attend(width=(most - 2) // page, page=page) == -1 and b"NULL" in h.dk_last_error()  # as far as the pointers
        assert attend(width=(most - 2) // page + 1, page=page) == -1 and b"2^31" in h.dk_last_error()
    assert attend(width=most // 16 - 100, T=2000) == -1 and b"2^31" in h.dk_last_error()
    for more in (dict(width=1 << 60), dict(pages=1 << 59), dict(pages=1 << 62), dict(window=1 << 31), dict(sinks=1 << 40)):
        assert attend(**more) == -1 and b"2^31" in h.dk_last_error(), more


def test_c_entries_take_a_step_without_sequences():
    """A call of no tokens, of no sequences too, does nothing; tokens without a sequence are refused."""
    from kernels import _lib

    h = _lib.lib()

    def attend(T, B, starts=0):
        return h.dk_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(0, 1536, 0, 0, 4, 16, 0, 0, 0, 2, 2, 0, starts, 0, 0, 1.0, 0, T, B, 12,
                                                                   2, 128, 0, 0, 0, 0))

    def append(T, B):
        return h.dk_paged_append(_lib.PAGED_APPEND_ARGS.pack(0, 0, 0, 0, 4, 16, 0, 2, 2, 0, 0, 0, 0, 1, 64, 10, 0, 0, T, B, 12, 2, 128,
                                                             0, 0))

    assert attend(0, 0) == attend(0, 0, starts=256) == attend(0, 3, starts=256) == 0
    assert append(0, 0) == 0
    assert attend(2, 0, starts=256) == append(2, 0) == -1 and attend(0, -1) == append(0, -1) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("B", [0, 3])
def test_a_step_without_tokens(B):
    from kernels.paged import paged_append, paged_attention, shared_prefix_attention

    c = Case([(1, 20)] * 3, prefix=16, spoil=False)
    starts = torch.zeros(B + 1, dtype=torch.int32, device="cuda") if B else None
    table, lengths, k, v = c.table[:B], c.lengths[:B], c.k.clone(), c.v.clone()
    cos, sin = _rope(64, 128)
    assert paged_append(c.q.new_zeros(0, 16 * 128), c.k, c.v, table, lengths, cos, sin, 12, 2, starts).shape == (0, 12, 128)
    assert torch.equal(c.k, k) and torch.equal(c.v, v)
    assert paged_attention(c.q[:0], c.k, c.v, table, lengths, starts).shape == (0, 12, 128)
    assert shared_prefix_attention(c.q[:0], c.k, c.v, c.prefix_table, 16, table, lengths, starts).shape == (0, 12, 128)


def _one_wide(c):
    """Layouts whose strides differ from the usual only where an extent is 1: one head, one column of pages, one row of angles."""
    q = torch.randn(1, c.T, c.hd).to(c.dtype).to(c.q.device).transpose(0, 1)  # [T, 1, hd], heads T * hd apart
    table = c.table[:, :1].t().contiguous().t()  # [B, 1], columns B apart
    cos, sin = torch.ones(1, c.hd // 2, device=c.q.device), torch.zeros(3, c.hd // 2, device=c.q.device).as_strided((1, c.hd // 2), (7, 1))
    return q, table, cos.as_strided(cos.shape, (5, 1)), sin


def test_strides_of_extent_one_are_not_looked_at():
    """They pass the checks of layouts; the CPU tensors are refused after those."""
    from kernels.logprobs import token_logprobs
    from kernels.paged import paged_append, paged_attention

    c = Case([(1, 1), (1, 1)], nq=1, nkv=1, spoil=False, device="cpu")
    q, table, cos, sin = _one_wide(c)
    for call in (lambda: paged_attention(q, c.k, c.v, c.table, c.lengths), lambda: paged_attention(c.q, c.k, c.v, table, c.lengths),
                 lambda: paged_append(torch.zeros(2, 3 * 128).half(), c.k, c.v, table, c.lengths, cos, sin, 1, 1),
                 lambda: token_logprobs(torch.zeros(2, 4).t()[:, :1].as_strided((2, 1), (1, 9)), torch.zeros(2, dtype=torch.long))):
        with pytest.raises(RuntimeError, match="CUDA device"):
            call()


@pytest.mark.gpu
def test_one_head_one_page_one_angle():
    from kernels.logprobs import token_logprobs
    from kernels.paged import paged_append, paged_attention

    c = Case([(1, 1), (1, 1), (1, 1)], nq=1, nkv=1, spoil=False)
    q, table, cos, sin = _one_wide(c)
    want = paged_attention(q.contiguous().view(3, 1, 128), c.k, c.v, c.table, c.lengths)
    assert torch.equal(paged_attention(q, c.k, c.v, table, c.lengths), want)
    qkv = torch.randn(3, 3 * 128, device="cuda").half()
    out = paged_append(qkv, c.k, c.v, table, c.lengths, cos, sin, 1, 1)
    assert torch.equal(out.view(3, 128), qkv[:, :128])  # an angle of zero
    lp = token_logprobs(torch.randn(2, 1, device="cuda").as_strided((2, 1), (1, 9)), torch.zeros(2, dtype=torch.long, device="cuda"))[0]
    assert not lp.any()


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 256)])
@pytest.mark.parametrize("sinks", [0, 3, 40])
def test_windows_wholly_past_the_table_leave_the_sinks(one_token, hd, page, sinks):
    """A length far past the table is reported; what counts is what the table has, here the sinks alone."""
    from kernels import _lib
    from kernels.paged import paged_attention

    c = Case([(1, 60), (1, 30)] if one_token else [(5, 60), (40, 45)], hd=hd, page=page, one_token=one_token, wide=0)
    for length in (c.table.shape[1] * page + 100, 2 ** 31 - 1):
        lengths = c.lengths.clone()
        lengths[0] = length
        _lib.clear_device_error()
        out = paged_attention(c.q, c.k, c.v, c.table, lengths, c.starts, window=20, sinks=sinks)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        exact, tol = c.attention(20, sinks)
        n = c.sizes[0][0]
        k, v, group = c.sequence(c.k, 0)[:sinks], c.sequence(c.v, 0)[:sinks], c.nq // c.nkv
        for t in range(n):  # over the positions 0..sinks - 1, with the tolerance of Case.attention
            if sinks == 0:
                exact[t], tol[t] = 0, 0
                continue
            a = torch.softmax(torch.einsum("hd,jhd->hj", c.q[t].double().cpu(), k.repeat_interleave(group, 1)) * hd ** -0.5, -1)
            vs = v.repeat_interleave(group, 1)
            exact[t] = torch.einsum("hj,jhd->hd", a, vs)
            u, spread = UNIT[c.dtype], torch.einsum("hj,jhd->hd", a, vs.abs())
            tol[t] = u * exact[t].abs() + (u + 2.0 ** -13) * spread + sinks * 2.0 ** -25 * vs.abs().max()
        assert_within(out, exact, tol)
