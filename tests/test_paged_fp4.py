"""The ops of a paged cache held in 4 bits (kernels.paged_fp4, C-ABI dk_paged_append_fp4, dk_paged_read_fp4, dk_paged_attention_fp4,
dk_shared_prefix_attention_fp4) against plain 64-bit implementations, at the sizes and masks where they can go wrong, and
their refusals."""

import math

import pytest
import torch

from _paged import UNIT, Case, assert_within
from _paged_fp4 import NUMBERS, SCALES, Fp4Case, pack, quantise, unpack

F16, BF16 = torch.float16, torch.bfloat16


# ------------------------------------------------------------------------------------------ the format, on the CPU
def test_the_format_written_twice():
    """The plain implementation of the tests and the one of the timed workloads agree, borders and odd values included."""
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("more_operators", Path(__file__).resolve().parents[1] / "perf" / "more_operators.py")
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    for dtype, power in ((F16, 1.0), (BF16, 0.25), (BF16, 2.0 ** 20)):
        x = _odd_values(dtype, power)
        codes, scales, values = quantise(x, power)
        packed, grid = ops._quantise(x, power)
        assert torch.equal(grid.long(), scales)
        assert torch.equal(torch.stack([packed % 16, packed // 16], -1).flatten(-2).long(), codes)
        assert torch.equal(ops._values(packed, grid, power).double(), values)
        pool = pack(codes.view(-1, 1, 2, x.shape[-1]), scales.view(-1, 1, 2, x.shape[-1] // 16))
        again = unpack(pool)
        assert torch.equal(again[0].flatten(), codes.flatten()) and torch.equal(again[1].flatten(), scales.flatten())


def _odd_values(dtype, power, dim=64, rows=400):
    """Rows of a 16-bit type whose ratios to their scales hit borders between codes, scales between scales; zeros, tiny and
    largest values, one value alone."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(rows, dim, generator=g, dtype=torch.float64)
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    for i in range(120):  # a scale with four bits of significand, values on and next to the borders
        unit = SCALES[8 + 7 * i % 100]
        row = border[torch.randint(0, 7, (dim,), generator=g)] * unit
        row[torch.rand(dim, generator=g) < 0.3] *= 1 + 2.0 ** -10
        row[torch.rand(dim, generator=g) < 0.3] *= 1 - 2.0 ** -10
        row[0::16] = 6 * unit
        x[i] = row * torch.where(torch.rand(dim, generator=g) < 0.5, -1.0, 1.0)
    for i in range(120, 180):  # largest values halfway between two scales
        x[i] *= 0.1
        x[i, 0::16] = 6 * (SCALES[i - 60] + SCALES[i - 59]) / 2
    x[180:200] = 0
    x[200:220] *= 2.0 ** -10 * torch.rand(20, 1, generator=g, dtype=torch.float64)
    x[220:230] *= 1e4
    x[230:240] = 0
    x[230:240, 5] = torch.linspace(0.001, 3000, 10, dtype=torch.float64)
    x[240] = torch.finfo(dtype).max / power
    x[241] = -0.0
    return (x * power).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)


# ------------------------------------------------------------------------------------------ append
def _rope(positions, hd, dtype=torch.float32):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()


def _appended(c, qkv, cos, sin, offset=0):
    """What appending qkv has to leave in the pools: (codes, scale bytes) of k and of v, from the pools before."""
    half, nq, nkv = c.hd // 2, c.nq, c.nkv
    x = qkv.cpu().view(-1, nq + 2 * nkv, c.hd)
    k, v = unpack(c.k_pool.cpu()), unpack(c.v_pool.cpu())
    t = 0
    for b, (new, n) in enumerate(c.sizes):
        for i in range(new):
            p = n - new + i
            if p >= 0:
                a, s = cos[p + offset].double().cpu(), sin[p + offset].double().cpu()
                lo, hi = x[t, nq:nq + nkv, :half].double(), x[t, nq:nq + nkv, half:].double()
                turned = torch.cat([lo * a - hi * s, hi * a + lo * s], -1).to(c.dtype)
                row, at = c.table[b, p // c.page].long().item(), p % c.page
                k[0][row, :, at], k[1][row, :, at], _ = quantise(turned, c.k_scale)
                v[0][row, :, at], v[1][row, :, at], _ = quantise(x[t, nq + nkv:], c.v_scale)
            t += 1
    return k, v


def _same(pool, want):
    codes, scales = unpack(pool.cpu())
    assert torch.equal(scales, want[1])
    real = (scales < 127).repeat_interleave(16, -1)  # a NaN scale says it all
    assert torch.equal(codes[real], want[0][real])


APPEND = [
    ([(1, 1)], 12, 2, 128, 16, F16, torch.float32, 0, 1.0, 1.0),
    ([(1, 17), (1, 300), (1, 64), (1, 65)], 28, 4, 128, 64, BF16, torch.float32, 0, 0.25, 2.0 ** -4),
    ([(5, 5), (0, 9), (33, 70), (1, 1), (100, 129)], 7, 1, 64, 32, F16, F16, 0, 1.0, 0.5),
    ([(3, 250), (129, 400)], 8, 8, 64, 256, BF16, BF16, 11, 2.0 ** 10, 2.0 ** -10),
    ([(1, 0), (1, 40), (1, -3)], 4, 1, 128, 128, F16, torch.float32, 1000, 4.0, 1.0),  # unused slots of the batch
    ([(300, 700)], 3, 3, 64, 16, F16, torch.float32, 0, 1.0, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,table_type,offset,k_scale,v_scale", APPEND)
def test_append(sizes, nq, nkv, hd, page, dtype, table_type, offset, k_scale, v_scale):
    from kernels import _lib
    from kernels.paged import paged_append
    from kernels.paged_fp4 import paged_append_fp4

    c = Fp4Case(sizes, nq, nkv, hd, page, dtype, spoil=False, k_scale=k_scale, v_scale=v_scale)
    qkv = torch.randn(c.T, nq + 2 * nkv, hd, device="cuda")
    qkv[:, nq:nq + nkv] *= 20 * k_scale
    qkv[:, nq + nkv:] *= v_scale
    wide = torch.zeros(c.T, (nq + 2 * nkv) * hd + 8, dtype=dtype, device="cuda")  # strided rows
    wide[:, :-8] = qkv.to(dtype).view(c.T, -1)
    qkv = wide[:, :-8]
    cos, sin = _rope(max(n for _, n in sizes) + offset + 1, hd, table_type)
    want_k, want_v = _appended(c, qkv.contiguous(), cos, sin, offset)
    _lib.clear_device_error()
    q = paged_append_fp4(qkv, c.k_pool, c.v_pool, c.table, c.lengths, cos, sin, nq, nkv, starts=c.starts, offset=offset, **c.scales)
    assert _lib.device_error() == 0
    _same(c.k_pool, want_k)  # nothing else in the pools changed either
    _same(c.v_pool, want_v)
    like = [torch.zeros(*c.k_pool.shape[:3], hd, dtype=dtype, device="cuda") for _ in range(2)]
    assert torch.equal(q, paged_append(qkv, *like, c.table, c.lengths, cos, sin, nq, nkv, starts=c.starts, offset=offset))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("power", [1.0, 2.0 ** -6, 2.0 ** 3])
def test_append_borders(dtype, power):
    """Values on the borders between codes and scales, zeros, tiny and largest ones, infinities and NaN, as k and as v: an angle
    of zero leaves k as it is."""
    from kernels.paged_fp4 import paged_append_fp4, paged_read_fp4

    x = _odd_values(dtype, power)
    x[250, 3], x[251, 20], x[252, 40], x[253, :] = math.inf, -math.inf, math.nan, math.inf
    T = x.shape[0]
    c = Fp4Case([(T, T)], nq=1, nkv=1, hd=64, page=16, dtype=dtype, spoil=False, k_scale=power, v_scale=power, one_token=False)
    qkv = torch.cat([x, x, x.flip(1)], -1).cuda()
    cos, sin = torch.ones(T, 32, device="cuda"), torch.zeros(T, 32, device="cuda")
    x[250:254] = torch.where(x[250:254].isinf() | x[250:254].isnan(), 0.0, x[250:254].float()).to(dtype)  # an infinity times sin 0 is NaN
    want = _appended(c, qkv, cos, sin)
    paged_append_fp4(qkv, c.k_pool, c.v_pool, c.table, c.lengths, cos, sin, 1, 1, starts=c.starts, **c.scales)
    _same(c.k_pool, want[0])
    _same(c.v_pool, want[1])
    k, v = paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, tokens=T, dtype=dtype, **c.scales)
    for got, value in ((k, quantise(qkv[:, 64:128].cpu(), power)[2]), (v, quantise(qkv[:, 128:].cpu(), power)[2])):
        clean = torch.ones(T, dtype=torch.bool)
        clean[250:254] = False  # (the rotation spreads those to the other half)
        assert torch.equal(got[:, 0].double().cpu()[clean], value.to(dtype).double()[clean])
    value = quantise(qkv[:, 128:].cpu(), power)[2].to(dtype).double()
    assert torch.equal(v[:, 0].double().cpu().nan_to_num(nan=12345.0), value.nan_to_num(nan=12345.0))


@pytest.mark.gpu
def test_append_without_a_page_or_an_angle_writes_nothing():
    from kernels import _lib
    from kernels.paged_fp4 import paged_append_fp4

    c = Fp4Case([(1, 20), (1, 5)], spoil=False)
    cos, sin = _rope(64, 128)
    qkv = torch.randn(2, 16 * 128, device="cuda").half()
    for spoil in ("table", "pool", "angle"):
        k, v, table = c.k_pool.clone(), c.v_pool.clone(), c.table.clone()
        table[:, :] = {"table": -1, "pool": c.k_pool.shape[0], "angle": 0}[spoil]
        rows = slice(0, 3) if spoil == "angle" else slice(0, 64)
        _lib.clear_device_error()
        paged_append_fp4(qkv, k, v, table, c.lengths, cos[rows], sin[rows], 12, 2)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        assert torch.equal(k, c.k_pool) and torch.equal(v, c.v_pool)


@pytest.mark.gpu
@pytest.mark.parametrize("before,after", [(0, 4), (2, 0), (1, 3)])
def test_append_and_read_rows_outside_starts(before, after):
    """Rows before starts[0] and from starts[B] on belong to no sequence: they append nothing, and q, k and v are zero."""
    from kernels import _lib
    from kernels.paged_fp4 import paged_append_fp4, paged_read_fp4

    c = Fp4Case([(3, 20), (2, 40), (1, 0)], nkv=2, spoil=False)
    c.table[2] = c.table[0]  # an unused slot with another sequence's pages still in its row
    cos, sin = _rope(200, 128)
    qkv = torch.randn(before + c.T + after, 16 * 128, device="cuda").half()
    want_k, want_v = c.k_pool.clone(), c.v_pool.clone()
    want = paged_append_fp4(qkv[before:before + c.T].contiguous(), want_k, want_v, c.table, c.lengths, cos, sin, 12, 2, starts=c.starts)
    _lib.clear_device_error()
    q = paged_append_fp4(qkv, c.k_pool, c.v_pool, c.table, c.lengths, cos, sin, 12, 2, starts=c.starts + before)
    assert _lib.device_error() == 0
    assert torch.equal(c.k_pool, want_k) and torch.equal(c.v_pool, want_v)
    k, v = paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts + before, tokens=len(qkv))
    for got, plain in ((q, want), *zip((k, v), paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, tokens=c.T))):
        assert torch.equal(got[before:before + c.T], plain)
        assert not got[:before].any() and not got[before + c.T:].any()
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------------------ read back
@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nkv,hd,page,dtype,k_scale,v_scale", [
    ([(1, 1)], 2, 128, 16, F16, 1.0, 1.0),
    ([(1, 40), (1, 0), (1, 129)], 4, 128, 64, BF16, 0.25, 8.0),
    ([(70, 70), (0, 5), (33, 100)], 1, 64, 32, F16, 1.0, 2.0 ** -6),
    ([(300, 300), (5, 3), (4, 0)], 8, 64, 256, BF16, 2.0 ** 40, 2.0 ** -40),
    ([(513, 513)], 3, 128, 128, F16, 0.5, 1.0),
    ([(333, 400), (1, 20)], 5, 128, 16, BF16, 1.0, 1.0),  # columns that do not fill the warps of a block,
    ([(700, 700), (2, 9)], 20, 128, 64, F16, 1.0, 0.5),  # more of them than warps
    ([(19500, 19500), (3, 1)], 1, 64, 256, BF16, 1.0, 1.0),  # whole batches of rows
    ([(5000, 5003), (1, 4)], 2, 128, 32, F16, 2.0, 1.0),
])
def test_read(sizes, nkv, hd, page, dtype, k_scale, v_scale):
    """Exactly what the codes stand for; rows before a sequence's first position are zero."""
    from kernels import _lib
    from kernels.paged_fp4 import paged_read_fp4

    c = Fp4Case(sizes, nkv, nkv, hd, page, dtype, seed=4, k_scale=k_scale, v_scale=v_scale)
    _lib.clear_device_error()
    got = paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, tokens=c.T, dtype=dtype, **c.scales)
    assert _lib.device_error() == 0
    t = 0
    for b, (new, n) in enumerate(sizes):
        for pool, out in zip((c.k, c.v), got):
            want = torch.cat([torch.zeros(max(0, new - max(n, 0)), nkv, hd, dtype=torch.float64), c.sequence(pool, b)[max(0, n - new):]])
            assert torch.equal(out[t:t + new].double().cpu(), want)
        t += new
    into = tuple(torch.full_like(x, math.nan) for x in got)
    paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, out=into, **c.scales)
    assert torch.equal(into[0], got[0]) and torch.equal(into[1], got[1])


@pytest.mark.gpu
def test_read_reports_positions_without_a_page():
    from kernels import _lib
    from kernels.paged_fp4 import paged_read_fp4

    c = Fp4Case([(20, 50), (3, 30)], spoil=False, wide=0)
    whole = paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, tokens=23)
    for entry in (-1, c.k_pool.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 35 // c.page] = entry
        _lib.clear_device_error()
        got = paged_read_fp4(c.k_pool, c.v_pool, table, c.lengths, c.starts, tokens=23)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        lost = torch.tensor([(30 + i) // c.page == 35 // c.page if i < 20 else False for i in range(23)], device="cuda")
        for x, y in zip(got, whole):
            assert not x[lost].any() and torch.equal(x[~lost], y[~lost])
    paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths + 1000, c.starts, tokens=23)
    assert _lib.device_error() == 3
    _lib.clear_device_error()


# ------------------------------------------------------------------------------------------ attention
def _attend(c, **more):
    from kernels.paged_fp4 import paged_attention_fp4

    return paged_attention_fp4(c.q, c.k_pool, c.v_pool, c.table, c.lengths, starts=c.starts, **{**c.scales, **more})


def _attend_prefix(c, **more):
    from kernels.paged_fp4 import shared_prefix_attention_fp4

    return shared_prefix_attention_fp4(c.q, c.k_pool, c.v_pool, c.prefix_table, c.prefix, c.table, c.lengths, starts=c.starts,
                                       **{**c.scales, **more})


ONE_TOKEN = [
    # sizes, nq, nkv, hd, page, dtype, window, sinks, k_scale, v_scale
    ([(1, 1)], 12, 2, 128, 16, F16, 0, 0, 1.0, 1.0),
    ([(1, 640)], 12, 2, 128, 16, F16, 0, 0, 0.25, 2.0 ** -4),
    ([(1, 63), (1, 64), (1, 65), (1, 1), (1, 0), (1, 129)], 28, 4, 128, 64, BF16, 0, 0, 1.0, 0.5),
    ([(1, 1000), (1, 3), (1, 517)], 16, 1, 128, 32, F16, 0, 0, 1.0, 1.0),
    ([(1, 700), (1, 31)], 8, 8, 64, 128, BF16, 0, 0, 4.0, 1.0),
    ([(1, 300)] * 70, 4, 1, 64, 16, F16, 0, 0, 1.0, 1.0),
    ([(1, 777), (1, 40), (1, 5)], 12, 2, 128, 16, F16, 100, 4, 1.0, 2.0 ** -8),
    ([(1, 777), (1, 40), (1, 128)], 14, 2, 128, 64, BF16, 1, 0, 1.0, 1.0),
    ([(1, 777), (1, 100)], 7, 1, 128, 32, F16, 64, 70, 2.0, 1.0),  # the sinks reach into the second chunk
    ([(1, 90), (1, 300)], 4, 2, 64, 16, F16, 1 << 30, 3, 1.0, 1.0),
    ([(1, 2000), (1, 130)], 9, 1, 64, 256, BF16, 0, 0, 1.0, 1.0),
    ([(1, 255), (1, 256), (1, 257)], 22, 2, 128, 256, F16, 0, 0, 1.0, 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,window,sinks,k_scale,v_scale", ONE_TOKEN)
def test_attention_one_token(sizes, nq, nkv, hd, page, dtype, window, sinks, k_scale, v_scale):
    from kernels import _lib

    c = Fp4Case(sizes, nq, nkv, hd, page, dtype, seed=1, k_scale=k_scale, v_scale=v_scale)
    _lib.clear_device_error()
    out = _attend(c, window=window, sinks=sinks)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, _attend(c, window=window, sinks=sinks))


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
    ([(4, 900), (2, 31), (5, 500), (1, 64), (3, 2)], 12, 2, 128, 32, BF16, 0, 0),  # drafted tokens
    ([(2, 700), (6, 333), (5, 90)], 4, 1, 64, 16, F16, 70, 3),
    ([(3, 700), (2, 333)], 14, 1, 128, 64, F16, 0, 0),
    ([(300, 500)] + [(0, 10)] * 15 + [(90, 90)], 12, 2, 128, 32, BF16, 0, 0),  # few tokens a slot: chunks converted for each tile
    ([(300, 500)] + [(0, 10)] * 15, 12, 2, 128, 64, F16, 130, 9),
    ([(200, 333)] + [(0, 0)] * 9, 6, 2, 64, 16, F16, 0, 0),
    ([(1, 700), (6, 90), (7, 90), (50, 400), (1, 0), (1, 1), (3, 333), (2, 2)], 12, 2, 128, 16, F16, 0, 0),  # decode beside prompts
    ([(1, 700), (6, 90), (7, 90), (500, 600), (1, 0), (1, 1), (3, 333), (2, 2)], 12, 2, 128, 16, BF16, 100, 3),
    ([(1, 257), (30, 100), (50, 60), (48, 300), (49, 300)], 2, 2, 64, 256, BF16, 0, 0),
    ([(4, 4)], 16, 2, 128, 16, F16, 0, 0),
    ([(200, 260), (4, 77), (180, 180), (150, 400)], 12, 2, 128, 16, BF16, 0, 0),  # prompts of several tiles: copied first
    ([(200, 260), (4, 77), (180, 180), (150, 400)], 28, 4, 64, 64, F16, 60, 5),
    ([(250, 300)], 16, 1, 128, 256, F16, 0, 0),
    ([(130, 500), (1, 0), (1, 9)], 14, 1, 128, 32, F16, 25, 17),
    ([(9, 7)], 4, 2, 64, 16, BF16, 3, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,window,sinks", RAGGED)
def test_attention_ragged(sizes, nq, nkv, hd, page, dtype, window, sinks):
    from kernels import _lib

    c = Fp4Case(sizes, nq, nkv, hd, page, dtype, seed=2, one_token=False, k_scale=0.5, v_scale=2.0)
    _lib.clear_device_error()
    out = _attend(c, window=window, sinks=sinks)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, _attend(c, window=window, sinks=sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,nq,nkv,hd,page,dtype,window,sinks", RAGGED + [
    ([(60, 700), (50, 120), (2, 100), (9, 9)], 8, 2, 64, 256, F16, 100, 5),
    ([(60, 700), (50, 120), (2, 100), (9, 9)], 12, 2, 128, 128, BF16, 100, 70),
    ([(9, 5), (40, 200), (3, 0)], 12, 2, 128, 16, F16, 1 << 30, 3),
    ([(70, 200), (3, 90)], 12, 2, 128, 32, BF16, 40, 2),
    ([(2, 40)] * 70 + [(30, 31)], 8, 4, 64, 16, BF16, 33, 1),
])
def test_attention_ragged_in_wide_tables(sizes, nq, nkv, hd, page, dtype, window, sinks):
    """Page tables so wide that the call might be a large one: split by the sequences' tokens between two kernels."""
    from kernels import _lib

    c = Fp4Case(sizes, nq, nkv, hd, page, dtype, seed=2, one_token=False, wide=1 << 16)
    _lib.clear_device_error()
    out = _attend_in(c, 1, window, sinks)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, _attend(c, window=window, sinks=sinks))


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

    c = Fp4Case(sizes, nq, nkv, hd, page, dtype, seed=7, prefix=prefix, k_scale=2.0, v_scale=0.25)
    _lib.clear_device_error()
    out = _attend_prefix(c)
    assert _lib.device_error() == 0
    assert_within(out, *c.attention())
    assert torch.equal(out, _attend_prefix(c))
    c.prefix = 0
    assert torch.equal(_attend_prefix(c), _attend(c))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq", [(128, 8), (64, 8), (128, 80)])
def test_attention_long_rings(hd, nq):
    """Many more chunks per CTA than its ring has slots, call after call without a host wait in between: every call gives
    the first one's bits, and no bounded wait gives up."""
    from kernels import _lib

    c = Fp4Case([(1, 4000 + 97 * b) for b in range(10)], nq=nq, nkv=8, hd=hd, page=64, seed=8, spoil=False)
    _lib.clear_device_error()
    first = _attend(c)
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(200):
        same &= (_attend(c) == first).all()
    assert same.item() and _lib.device_error() == 0
    few = Fp4Case([(1, 4000 + 97 * b) for b in range(2)], nq=nq, nkv=8, hd=hd, page=64, seed=9)
    assert_within(_attend(few), *few.attention())


def _attend_in(c, fill, window=0, sinks=0):
    """The call's output, made in a workspace that holds `fill` in each of its 32-bit words."""
    import ctypes

    from kernels import _lib
    from kernels.paged import _DTYPES

    T, B, code, width = c.q.shape[0], c.lengths.numel(), _DTYPES[c.dtype], c.table.shape[1]
    n, prefix = ctypes.c_uint64(0), c.prefix if c.prefix else 0
    _lib.call("dk_paged_attention_fp4_workspace_bytes", T, B, c.nq, c.nkv, c.hd, code, c.starts is not None, prefix, width * c.page,
              ctypes.byref(n))
    ws = torch.full((n.value // 4,), fill, dtype=torch.int32, device="cuda")
    out = torch.full((T, c.nq, c.hd), torch.nan, dtype=c.dtype, device="cuda")
    args = _lib.PAGED_ATTENTION_FP4_ARGS.pack(
        c.q.data_ptr(), c.q.stride(0), c.k_pool.data_ptr(), c.v_pool.data_ptr(), c.k_pool.shape[0], c.page,
        c.prefix_table.data_ptr() if prefix else 0, prefix, c.table.data_ptr(), c.table.stride(0), width, c.lengths.data_ptr(),
        0 if c.starts is None else c.starts.data_ptr(), window, sinks, c.hd ** -0.5, out.data_ptr(), T, B, c.nq, c.nkv, c.hd, code,
        ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream, c.scales["k_scale"], c.scales["v_scale"])
    entry = "dk_shared_prefix_attention_fp4" if prefix else "dk_paged_attention_fp4"
    _lib.check(getattr(_lib.lib(), entry)(args), entry)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("sizes,prefix", [
    ([(2, 40)] * 70, 0),  # as many units of tiles as CTAs may come, none does
    ([(1, 900), (2, 40)] * 40, 0),
    ([(2, 40)] * 69 + [(60, 300)], 0),
    ([(3, 40)] * 4, 0),
    ([(1, 500)], 0),
    ([(1, 33)] * 300, 0),
    ([(130, 400), (7, 9), (1, 3000)], 0),
    ([(600, 900), (500, 600)], 0),  # copied
    ([(1, 40)] * 20, 300),
    ([(2, 40), (90, 100)] * 10, 300),
])
def test_workspaces_may_hold_anything(sizes, prefix, dtype, hd):
    """What a workspace held before a call changes nothing of it: not zeros, nor NaN, nor words that could be records of
    the call's own."""
    c = Fp4Case(sizes, nq=8, nkv=4, hd=hd, page=16, dtype=dtype, prefix=prefix, seed=11)
    out = _attend_in(c, 1)
    assert_within(out, *c.attention())
    assert torch.equal(out, _attend_in(c, 0)) and torch.equal(out, _attend_in(c, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv,dtype,page", [(128, 28, 4, BF16, 16), (64, 6, 2, F16, 256), (128, 9, 1, BF16, 64)])
@pytest.mark.parametrize("sizes,window,sinks", [
    ([(1, 1)], 0, 0),
    ([(1, 0), (1, 256), (1, 200), (1, 0)], 0, 0),
    ([(1, 1 + 7 * b % 384) for b in range(150)], 0, 0),  # more units than groups, or fewer
    ([(1, 640 - b) for b in range(56)], 0, 0),
    ([(1, 1500), (1, 3), (1, 90)], 60, 5),  # short windows over long caches
    ([(1, 1500), (1, 3), (1, 90)] * 20, 130, 140),
    ([(2, 300), (0, 0), (1, 20), (3, 2)], 0, 0),
    ([(2, 900), (0, 10), (1, 20), (2, 1)], 33, 1),
])
def test_attention_of_short_units(sizes, window, sinks, hd, nq, nkv, dtype, page):
    """Short page tables and short windows: no sequence's work is cut."""
    c = Fp4Case(sizes, nq=nq, nkv=nkv, hd=hd, page=page, dtype=dtype, seed=12)
    out = _attend_in(c, 1, window, sinks)
    assert_within(out, *c.attention(window, sinks))
    assert torch.equal(out, _attend(c, window=window, sinks=sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,dtype", [(64, BF16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("sizes", [
    [(900, 2500), (300, 1500)],  # copied, 16-bit tiles
    [(400, 6000), (90, 3000)] + [(0, 0)] * 30,  # tiles that convert for themselves
    [(5, 4000 + 97 * b) for b in range(10)],  # tiles of 16 rows
    [(2, 3000), (60, 5000), (3, 2000), (1, 4000), (50, 100)],  # both
])
def test_ragged_long_rings(sizes, hd, dtype):
    """Many more chunks than a ring has slots, call after call: the same bits, no wait that gives up, and the first call right."""
    from kernels import _lib

    c = Fp4Case(sizes, nq=6, nkv=2, hd=hd, page=32, seed=8, spoil=False, dtype=dtype)
    _lib.clear_device_error()
    first = _attend(c)
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(100):
        same &= (_attend(c) == first).all()
    assert same.item() and _lib.device_error() == 0
    if sum(n for n, _ in sizes) < 600:
        assert_within(first, *c.attention())


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
def test_attention_leaves_freed_pages_alone(one_token):
    """Pages outside the window and the sinks may be freed: their table entries point nowhere."""
    sizes = [(1, 700), (1, 130)] if one_token else [(9, 700), (40, 130)]
    c = Fp4Case(sizes, seed=3, one_token=one_token)
    window, sinks = 50, 4
    want = c.attention(window, sinks)
    for b, (new, n) in enumerate(sizes):
        first, last = 1, (n - new + 1 - window) // c.page
        for i in range(first, last):
            page = c.table[b, i].long().item()
            c.k_pool[page], c.v_pool[page] = 0x7f, 0x7f
        c.table[b, first:last] = torch.tensor([-1, 1 << 30]).repeat(last)[:last - first].int()
    assert_within(_attend(c, window=window, sinks=sinks), *want)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,window,sinks", [([(1, 400), (1, 31)], 0, 0), ([(70, 200), (3, 90)], 40, 2)])
def test_attention_strides_scale_stream_and_graph(sizes, window, sinks):
    """q rows inside a wider tensor, a table with spare columns, another scale, a side stream, a captured call."""
    from kernels.paged_fp4 import paged_attention_fp4

    c = Fp4Case(sizes, seed=4, k_scale=0.5, v_scale=4.0)
    wide = torch.zeros(c.T, c.nq + 5, c.hd, dtype=c.dtype, device="cuda")
    wide[:, :c.nq] = c.q
    table = torch.full((len(sizes), c.table.shape[1] + 40), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    args = (wide[:, :c.nq], c.k_pool, c.v_pool, table[:, :c.table.shape[1] + 3], c.lengths)
    more = dict(starts=c.starts, window=window, sinks=sinks, scale=0.2, **c.scales)
    want = c.attention(window, sinks, scale=0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = paged_attention_fp4(*args, **more)
    torch.cuda.current_stream().wait_stream(side)
    assert_within(out, *want)
    graph, kept = torch.cuda.CUDAGraph(), torch.empty_like(out)
    with torch.cuda.graph(graph):
        paged_attention_fp4(*args, out=kept, **more)
    graph.replay()
    assert torch.equal(kept, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("one_token", [True, False])
@pytest.mark.parametrize("size", [2.0 ** -8, 1.0, 60.0])
def test_attention_of_queries_of_any_size(dtype, one_token, size):
    """Scores far apart and all alike; queries whose heads differ by orders of magnitude, one of them zero. Beside Case.attention's
    terms: a score is a sum of 128 exact products in eight steps of fp32, each cutting off less than 2^-23 of sum |q| |k|, so it
    is off by up to 2^-20 of that, and so are the weights, above and below the division."""
    c = Fp4Case([(1, 3000), (1, 200)] if one_token else [(3, 700), (140, 300)], nq=6, nkv=2, dtype=dtype, seed=5, one_token=one_token)
    c.q *= size
    c.q[0, 0] *= 2.0 ** -12
    c.q[0, 1] = 0
    exact, tol = c.attention()
    group, t = c.nq // c.nkv, 0
    for b, (new, n) in enumerate(c.sizes):
        k, v = c.sequence(c.k, b).abs().repeat_interleave(group, 1), c.sequence(c.v, b).abs().amax(0).repeat_interleave(group, 0)
        for i in range(new):
            see = n - new + i + 1
            most = torch.einsum("hd,jhd->hj", c.q[t].double().cpu().abs(), k[:see]).amax(-1) * c.hd ** -0.5
            tol[t] += (2.0 ** -19 * most)[:, None] * v
            t += 1
    assert_within(_attend(c), exact, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[(1, 300)], [(1, 300), (1, 0), (1, 31)], [(9, 5), (4, 200), (3, 0)]])
def test_attention_windows_past_every_position(sizes):
    """A window as long as the table or longer masks nothing, up to the largest; rows before the first position are empty."""
    c = Fp4Case(sizes, one_token=all(n == 1 for n, _ in sizes))
    plain = _attend(c)
    assert_within(plain, *c.attention())
    for window in (c.table.shape[1] * c.page, 2 ** 31 - 1):
        for sinks in (0, 4, 2 ** 31 - 1):
            assert torch.equal(_attend(c, window=window, sinks=sinks), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 128, 256])
@pytest.mark.parametrize("sizes", [[(1, 700), (1, 101), (1, 100), (1, 3)], [(60, 700), (50, 120), (2, 100), (9, 9)]])
def test_attention_sinks_beside_the_window(page, sizes):
    """Sinks that end in their page, at its end, just before the window's first page, in it and beyond: the positions between
    are skipped, not seen."""
    c = Fp4Case(sizes, nq=4, nkv=2, hd=64, page=page)
    for sinks in (0, 1, 16, 17, 64, 256, 511, 512, 513, 599, 600, 690):
        assert_within(_attend(c, window=100, sinks=sinks), *c.attention(window=100, sinks=sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("sizes,prefix", [([(1, 9000)], 0), ([(5, 9000)], 0), ([(3, 5000), (70, 6000), (1, 40)], 0),
                                          ([(1, 3), (1, 700)], 9000), ([(4, 9), (30, 2000)], 5001)])
def test_units_cut_into_many_pieces(sizes, prefix, dtype, hd):
    """Few rows over long caches: every CTA works on the same units, whose many partial results are joined."""
    c = Fp4Case(sizes, nq=6, nkv=2, hd=hd, page=32, dtype=dtype, prefix=prefix)
    assert_within(_attend_prefix(c) if prefix else _attend(c), *c.attention())


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
def test_one_token_of_any_stride(ragged):
    """The row stride of a single token means nothing, whatever it is."""
    from kernels.paged_fp4 import paged_append_fp4

    c = Fp4Case([(1, 77)], one_token=not ragged)
    c.q = c.q.as_strided(c.q.shape, (3, c.hd, 1))
    assert_within(_attend(c), *c.attention())
    qkv = torch.randn(1, (c.nq + 2 * c.nkv) * c.hd, device="cuda", dtype=c.dtype)
    cos, sin = _rope(100, c.hd)
    pools = [(c.k_pool.clone(), c.v_pool.clone()) for _ in range(2)]
    a = paged_append_fp4(qkv, *pools[0], c.table, c.lengths, cos, sin, c.nq, c.nkv, c.starts)
    b = paged_append_fp4(qkv.as_strided(qkv.shape, (5, 1)), *pools[1], c.table, c.lengths, cos, sin, c.nq, c.nkv, c.starts)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(*pools))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 128), (BF16, 64)])
@pytest.mark.parametrize("scale", [0.0, -0.15, 1e-60])
@pytest.mark.parametrize("sizes,prefix,window,sinks", [
    ([(1, 200), (1, 3)], 0, 0, 0), ([(60, 300), (9, 9), (4, 2)], 0, 0, 0), ([(140, 400), (1, 90)], 0, 50, 3),
    ([(1, 70), (1, 0)], 200, 0, 0), ([(5, 30), (50, 60)], 333, 0, 0),
])
def test_scale_of_any_sign(sizes, prefix, window, sinks, scale, dtype, hd):
    """A scale of zero weighs the visible positions alike, a negative one the smallest products most (1e-60 is zero in fp32);
    masked positions stay out of it."""
    c = Fp4Case(sizes, nq=6, nkv=2, hd=hd, page=32, dtype=dtype, prefix=prefix, seed=10)
    exact, tol = c.attention(window, sinks, scale=scale)
    got = _attend_prefix(c, scale=scale) if prefix else _attend(c, window=window, sinks=sinks, scale=scale)
    assert_within(got, exact, tol)


def _without_prefix(c, q):
    """Case.attention of c's sequences with the queries q, as if there were no prefix."""
    kept = c.q, c.prefix
    c.q, c.prefix = q, 0
    got = c.attention()
    c.q, c.prefix = kept
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("before,after,hd", [(0, 700, 128), (2, 0, 64), (3, 5, 128)])
@pytest.mark.parametrize("sizes", [[(3, 20), (150, 200), (1, 0)], [(3, 20), (2, 200), (1, 0)]])
def test_attention_rows_outside_starts(before, after, hd, sizes):
    """Rows before starts[0] and from starts[B] on belong to no sequence: zero from attention over the pages, the prefix alone
    from attention with a prefix."""
    c = Fp4Case(sizes, hd=hd, one_token=False, prefix=40)
    own, live = c.q, slice(before, before + c.T)
    c.q = torch.cat([torch.randn(before, c.nq, hd), torch.zeros(c.T, c.nq, hd), torch.randn(after, c.nq, hd)]).to(c.dtype).cuda()
    c.q[live] = own
    outside = torch.ones(len(c.q), dtype=torch.bool)
    outside[live] = False
    exact, tol = _without_prefix(c, own)
    c.starts = c.starts + before
    out = torch.full_like(c.q, math.nan)
    _attend(c, out=out)
    assert_within(out[live], exact, tol)
    assert not out[outside.cuda()].any()
    out = torch.full_like(c.q, math.nan)
    _attend_prefix(c, out=out)
    alone = Fp4Case([(1, 0)] * int(outside.sum()), hd=hd, prefix=40)
    alone.q, alone.k, alone.v, alone.prefix_table = c.q[outside.cuda()], c.k, c.v, c.prefix_table
    assert_within(out[outside.cuda()], *alone.attention())


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
@pytest.mark.parametrize("window", [0, 30])
def test_attention_reports_positions_without_a_page(one_token, window):
    """A visible position whose table entry names no page of the pool counts as zeros and sets the device error, as does a length
    past the table; an entry that no row sees does not."""
    from kernels import _lib

    c = Fp4Case([(1, 200), (1, 50)] if one_token else [(40, 200), (3, 50)], one_token=one_token, spoil=False, prefix=100, wide=0)
    page, prefix = c.page, c.prefix

    def error(table=None, lengths=None, prefix_table=None, want=None):
        keep = c.table, c.lengths, c.prefix_table
        c.table, c.lengths = keep[0] if table is None else table, keep[1] if lengths is None else lengths
        _lib.clear_device_error()
        out = _attend(c, window=window, sinks=2)
        code = _lib.device_error()
        if want is not None:
            assert_within(out, *want)
        if window == 0:
            _lib.clear_device_error()
            c.prefix_table = keep[2] if prefix_table is None else prefix_table
            _attend_prefix(c)
            assert _lib.device_error() == (code if prefix_table is None else 3)
        _lib.clear_device_error()
        c.table, c.lengths, c.prefix_table = keep
        return code

    assert error() == 0
    c.prefix = 0
    k, v = c.k.clone(), c.v.clone()
    lost = c.table[0, 190 // page].long().item()
    c.k[lost], c.v[lost] = 0, 0
    zeroed = c.attention(window, 2)
    c.k, c.v, c.prefix = k, v, prefix
    for entry in (-1, c.k_pool.shape[0], 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 190 // page] = entry
        assert error(table, want=zeroed) == 3  # DK_DEVERR_BAD_POSITION
        table = c.table.clone()
        table[1, 50 // page + 1:] = entry  # after the second sequence's last position
        assert error(table) == 0
        if window == 0:
            wrong = c.prefix_table.clone()
            wrong[2] = entry
            error(prefix_table=wrong)
    assert error(lengths=c.lengths + torch.tensor([table.shape[1] * page - 200 + 1, 0], dtype=torch.int32, device="cuda")) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("window", [0, 20])
def test_unused_slots_of_any_negative_length(ragged, window):
    """A length of the type's lowest value is an unused slot like any other <= 0."""
    from kernels import _lib
    from kernels.paged_fp4 import paged_append_fp4, paged_read_fp4

    c = Fp4Case([(3, 40), (3, 0), (2, 20), (3, 0)] if ragged else [(1, 40), (1, 0), (1, 20), (1, 0)], one_token=not ragged, spoil=False)
    low = torch.tensor([40, -2 ** 31, 20, -2 ** 31 + 2], dtype=torch.int32, device="cuda")
    cos, sin = _rope(64, 128)
    qkv = torch.randn(c.T, 16 * 128, device="cuda").half()
    _lib.clear_device_error()
    got = []
    for lengths in (c.lengths, low):
        k, v = c.k_pool.clone(), c.v_pool.clone()
        c.lengths = lengths
        out = _attend(c, window=window, sinks=2)
        q = paged_append_fp4(qkv, k, v, c.table, lengths, cos, sin, 12, 2, starts=c.starts)
        got.append((out, q, k, v, *paged_read_fp4(k, v, c.table, lengths, c.starts, tokens=c.T)))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B", [0, 3])
def test_a_step_without_tokens(B):
    from kernels.paged_fp4 import paged_append_fp4, paged_read_fp4

    c = Fp4Case([(1, 20)] * 3, prefix=16, spoil=False)
    c.starts = torch.zeros(B + 1, dtype=torch.int32, device="cuda") if B else None
    c.table, c.lengths, c.q, k, v = c.table[:B], c.lengths[:B], c.q[:0], c.k_pool.clone(), c.v_pool.clone()
    cos, sin = _rope(64, 128)
    assert paged_append_fp4(c.q.new_zeros(0, 16 * 128), c.k_pool, c.v_pool, c.table, c.lengths, cos, sin, 12, 2, c.starts).shape == (0, 12, 128)
    assert torch.equal(c.k_pool, k) and torch.equal(c.v_pool, v)
    assert _attend(c).shape == (0, 12, 128) and _attend_prefix(c).shape == (0, 12, 128)
    assert [x.shape for x in paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, c.starts, tokens=0)] == [(0, 2, 128)] * 2


@pytest.mark.gpu
@pytest.mark.parametrize("one_token", [True, False])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 256)])
@pytest.mark.parametrize("sinks", [0, 3, 40])
def test_windows_wholly_past_the_table_leave_the_sinks(one_token, hd, page, sinks):
    """A length far past the table is reported; what counts is what the table has, here the sinks alone."""
    from kernels import _lib

    c = Fp4Case([(1, 60), (1, 30)] if one_token else [(5, 60), (40, 45)], hd=hd, page=page, one_token=one_token, wide=0)
    own = c.lengths
    for length in (c.table.shape[1] * page + 100, 2 ** 31 - 1):
        c.lengths = own.clone()
        c.lengths[0] = length
        _lib.clear_device_error()
        out = _attend(c, window=20, sinks=sinks)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        exact, tol = c.attention(20, sinks)
        k, v, group = c.sequence(c.k, 0)[:sinks], c.sequence(c.v, 0)[:sinks], c.nq // c.nkv
        for t in range(c.sizes[0][0]):  # over the positions 0..sinks - 1, with the tolerance of Case.attention
            if sinks == 0:
                exact[t], tol[t] = 0, 0
                continue
            a = torch.softmax(torch.einsum("hd,jhd->hj", c.q[t].double().cpu(), k.repeat_interleave(group, 1)) * hd ** -0.5, -1)
            vs = v.repeat_interleave(group, 1)
            exact[t] = torch.einsum("hj,jhd->hd", a, vs)
            u, spread = UNIT[c.dtype], torch.einsum("hj,jhd->hd", a, vs.abs())
            tol[t] = u * exact[t].abs() + (u + 2.0 ** -13) * spread + sinks * 2.0 ** -25 * vs.abs().max()
        assert_within(out, exact, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("sizes", [[(1, 90), (1, 70)], [(5, 90), (4, 70)], [(150, 200), (140, 140)], [(40, 200), (35, 140)]])
def test_a_nan_reaches_the_rows_that_see_it(sizes, dtype, hd):
    """A NaN scale at a visible position makes the results of its kv head NaN, in its sequence only. (Every row of the first sequence
    sees its position 3; one token each, few and many of them run different kernels.)"""
    for pool in ("k_pool", "v_pool"):
        c = Fp4Case(sizes, nq=4, nkv=2, hd=hd, page=16, dtype=dtype, seed=12)
        flat = getattr(c, pool)[c.table[0, 0].long(), 1].view(-1)  # kv head 1 of the first page
        flat[16 * hd // 2 + 3 * hd // 16] = 0x7f
        out = _attend(c)
        n = sizes[0][0]
        bad = out[:n, 2:].isnan()
        assert bad.all() if pool == "k_pool" else bad[..., :16].all() and not bad[..., 16:].any()
        assert out[:n, :2].isfinite().all() and out[n:].isfinite().all()


@pytest.mark.gpu
def test_pools_off_their_alignment_are_refused():
    from kernels.paged_fp4 import paged_append_fp4, paged_attention_fp4, paged_read_fp4

    c = Fp4Case([(1, 20)], spoil=False)
    room = torch.zeros(c.k_pool.numel() + 16, dtype=torch.uint8, device="cuda")
    odd = room[8:8 + c.k_pool.numel()].view(c.k_pool.shape)
    cos, sin = _rope(64, 128)
    qkv = torch.zeros(1, 16 * 128, device="cuda").half()
    for k, v in ((odd, c.v_pool), (c.k_pool, odd)):
        for call in (lambda: paged_attention_fp4(c.q, k, v, c.table, c.lengths), lambda: paged_read_fp4(k, v, c.table, c.lengths),
                     lambda: paged_append_fp4(qkv, k, v, c.table, c.lengths, cos, sin, 12, 2)):
            with pytest.raises(RuntimeError, match="alignment"):
                call()


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Each call has a workspace of its own: calls side by side give what they give alone."""
    cases = [Fp4Case([(1, 900 + 50 * b) for b in range(6)], seed=20, spoil=False), Fp4Case([(3, 700), (140, 300), (1, 50)], seed=21, spoil=False),
             Fp4Case([(200, 1200), (260, 700)], seed=22, dtype=BF16, spoil=False), Fp4Case([(1, 40), (1, 90)], seed=23, prefix=600, spoil=False)]
    run = [_attend, _attend, _attend, _attend_prefix]
    want = [f(c) for f, c in zip(run, cases)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    same = []
    for _ in range(20):
        for f, c, s, w in zip(run, cases, streams, want):
            with torch.cuda.stream(s):
                same.append((f(c) == w).all())
    torch.cuda.synchronize()
    assert torch.stack(same).all()


# ------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
def test_a_run_of_them_together(dtype, hd):
    """A prompt in two chunks and three decode steps of two sequences, all through the ops, against 64 bits on the values that the
    definition of the cache gives; the steps again behind a shared prefix; all of it once more from a captured graph."""
    from kernels.paged_fp4 import fp4_pages, paged_append_fp4, paged_attention_fp4, paged_read_fp4, shared_prefix_attention_fp4

    nq, nkv, page, prompt, steps = 6, 2, 16, [50, 75], 3
    scales = {"k_scale": 0.5, "v_scale": 0.25}
    g = torch.Generator().manual_seed(11)
    total = [n + steps for n in prompt]
    x = [torch.randn(n, (nq + 2 * nkv) * hd, generator=g).to(dtype) for n in total]
    cos, sin = _rope(max(total) + 1, hd)
    width = -(-max(total) // page)
    table = torch.randperm(2 * width, generator=g).int().view(2, width).cuda()
    # what every position holds, and what every row of the run has to give
    want, queries = [], []
    for b in range(2):
        rows = x[b].view(-1, nq + 2 * nkv, hd)
        a, s = cos[:total[b]].double().cpu()[:, None], sin[:total[b]].double().cpu()[:, None]
        lo, hi = rows[:, :nq + nkv, :hd // 2].double(), rows[:, :nq + nkv, hd // 2:].double()
        turned = torch.cat([lo * a - hi * s, hi * a + lo * s], -1)
        k = quantise(turned[:, nq:].to(dtype), scales["k_scale"])[2]
        v = quantise(rows[:, nq + nkv:], scales["v_scale"])[2]
        queries.append((turned[:, :nq], k, v))
        p = torch.einsum("thd,jhd->htj", turned[:, :nq], k.repeat_interleave(nq // nkv, 1)) * hd ** -0.5
        p = p.masked_fill(torch.arange(total[b])[None] > torch.arange(total[b])[:, None], -math.inf).softmax(-1)
        vs = v.repeat_interleave(nq // nkv, 1)
        spread = torch.einsum("htj,jhd->thd", p, vs.abs())
        out = torch.einsum("htj,jhd->thd", p, vs)
        # beside Case.attention's terms: q is rounded to the type first, which moves a score by u sum |q| |k|
        move = UNIT[dtype] * torch.einsum("thd,jhd->thj", turned[:, :nq].abs(), k.abs().repeat_interleave(nq // nkv, 1)).amax(-1) * hd ** -0.5
        tol = UNIT[dtype] * out.abs() + (UNIT[dtype] + 2.0 ** -13 + 2.5 * move[..., None]) * spread + total[b] * 2.0 ** -25 * vs.abs().max()
        want.append((out, tol))
    pools = [fp4_pages(2 * width, nkv, page, hd, "cuda") for _ in range(2)]

    def call(sizes, attend):
        """Appends and attends to `sizes` = [(tokens, positions)] of the two sequences."""
        one = all(n == 1 for n, _ in sizes)
        starts = None if one else torch.tensor([0, sizes[0][0], sizes[0][0] + sizes[1][0]], dtype=torch.int32, device="cuda")
        lengths = torch.tensor([n for _, n in sizes], dtype=torch.int32, device="cuda")
        qkv = torch.cat([x[b][n - new:n] for b, (new, n) in enumerate(sizes)]).cuda()
        q = paged_append_fp4(qkv, *pools, table, lengths, cos, sin, nq, nkv, starts, **scales)
        return attend(q, lengths, starts)

    plain = lambda q, lengths, starts: paged_attention_fp4(q, *pools, table, lengths, starts, **scales)  # noqa: E731
    chunks = [[(30, 30), (40, 40)], [(20, 50), (35, 75)]] + [[(1, n + i + 1) for n in prompt] for i in range(steps)]
    eager = []
    for sizes in chunks:
        out, t = call(sizes, plain), 0
        eager.append(out)
        for b, (new, n) in enumerate(sizes):
            assert_within(out[t:t + new], want[b][0][n - new:n], want[b][1][n - new:n])
            t += new
    ends = torch.tensor(total, dtype=torch.int32, device="cuda")
    k, v = paged_read_fp4(*pools, table, ends, torch.tensor([0, total[0], sum(total)], dtype=torch.int32, device="cuda"),
                          tokens=sum(total), dtype=dtype, **scales)
    assert torch.equal(k.double().cpu(), torch.cat([queries[b][1] for b in range(2)]))
    assert torch.equal(v.double().cpu(), torch.cat([queries[b][2] for b in range(2)]))
    # behind a shared prefix: the first sequence's first two pages before its own later ones give the same rows
    q0 = queries[0][0][-1:].to(dtype).cuda()
    own = table[:1, 2:].contiguous()
    got = shared_prefix_attention_fp4(q0, *pools, table[0], 32, own, ends[:1] - 32, **scales)
    assert_within(got, want[0][0][-1:], want[0][1][-1:])
    # one captured step serves all of them: the lengths and the tokens are read on the device
    lengths, qkv = torch.tensor(prompt, dtype=torch.int32, device="cuda"), torch.zeros(2, (nq + 2 * nkv) * hd, dtype=dtype, device="cuda")
    graph, kept = torch.cuda.CUDAGraph(), torch.empty(2, nq, hd, dtype=dtype, device="cuda")
    with torch.cuda.graph(graph):
        q = paged_append_fp4(qkv, *pools, table, lengths, cos, sin, nq, nkv, **scales)
        paged_attention_fp4(q, *pools, table, lengths, out=kept, **scales)
    for i in range(steps):
        lengths += 1
        qkv.copy_(torch.stack([x[b][prompt[b] + i] for b in range(2)]))
        graph.replay()
        assert torch.equal(kept, eager[2 + i])


# ------------------------------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    """Extents, types and layouts the kernels cannot take are refused before any device work."""
    from kernels.paged_fp4 import fp4_pages, paged_append_fp4, paged_attention_fp4, paged_read_fp4, shared_prefix_attention_fp4

    c = Fp4Case([(1, 20), (1, 5)], spoil=False, device="cpu")
    args = [c.q, c.k_pool, c.v_pool, c.table, c.lengths]
    starts = torch.tensor([0, 1, 2], dtype=torch.int32)
    assert fp4_pages(3, 2, 16, 128).shape == (3, 2, 16, 72) and fp4_pages(3, 2, 16, 64).shape == (3, 2, 16, 36)
    with pytest.raises(ValueError):
        fp4_pages(3, 2, 16, 96)

    def attend(error, *at, **more):
        a = list(args)
        for i, x in at:
            a[i] = x
        with pytest.raises(error):
            paged_attention_fp4(*a, **more)

    attend(RuntimeError)  # on the CPU
    attend(ValueError, (0, c.q[:1]))  # a token per sequence
    attend(ValueError, (0, c.q[..., :64]))
    attend(ValueError, (0, c.q[:, :5]))  # 5 query heads over 2 kv heads
    attend(ValueError, (0, torch.zeros(2, 34, 128).half()))  # 17 query heads for each kv head
    attend(ValueError, (0, c.q[:1].expand(2, -1, -1)))  # overlapping tokens
    attend(ValueError, (1, c.k_pool[:, :, :8].contiguous()), (2, c.v_pool[:, :, :8].contiguous()))
    attend(ValueError, (1, c.k_pool[:-1]))
    attend(ValueError, (1, c.k_pool.transpose(0, 1)), (2, c.v_pool.transpose(0, 1)))
    attend(ValueError, (1, c.k_pool[..., :64].contiguous()), (2, c.v_pool[..., :64].contiguous()))  # no whole position
    attend(ValueError, (3, c.table[:1]))
    attend(ValueError, (4, c.lengths[:1]))
    attend(ValueError, starts=starts[:2])
    attend(ValueError, window=-1)
    attend(ValueError, sinks=-1)
    attend(ValueError, out=torch.zeros(2, 12, 64).half())
    attend(RuntimeError, (0, c.q.float()))
    attend(RuntimeError, (1, c.k_pool.char()), (2, c.v_pool.char()))
    attend(RuntimeError, (2, c.v_pool.char()))
    attend(RuntimeError, (3, c.table.long()))
    for bad in (0.0, -1.0, 3.0, 1.5, math.inf, math.nan, 2.0 ** 65, 2.0 ** -65):
        attend(ValueError, k_scale=bad)
        attend(ValueError, v_scale=bad)
    attend(ValueError, k_scale=torch.ones(()))  # a number, not a tensor whose value may change
    for k in (1, 2.0 ** -64, 2.0 ** 64):
        attend(RuntimeError, k_scale=k)  # as far as the device
    for table, n in ((c.table[0], 1000), (c.table[0], -1)):
        with pytest.raises(ValueError):
            shared_prefix_attention_fp4(c.q, c.k_pool, c.v_pool, table, n, c.table, c.lengths)

    def read(error, **more):
        with pytest.raises(error):
            paged_read_fp4(c.k_pool, c.v_pool, c.table, c.lengths, **more)

    read(RuntimeError)  # on the CPU
    read(ValueError, tokens=3)  # one row per sequence
    read(ValueError, starts=starts)  # how many rows?
    read(ValueError, starts=starts, tokens=-1)
    read(ValueError, k_scale=3.0)
    read(RuntimeError, dtype=torch.float32)
    read(ValueError, out=(torch.zeros(2, 2, 128).half(), torch.zeros(2, 2, 128).bfloat16()))
    read(ValueError, out=(torch.zeros(2, 2, 64).half(), torch.zeros(2, 2, 64).half()))

    qkv, cos = torch.zeros(2, 16 * 128).half(), torch.zeros(40, 64)
    good = dict(qkv=qkv, cos=cos, sin=cos, n_heads=12, n_kv=2)

    def append(error, **more):
        a = {**good, **more}
        with pytest.raises(error):
            paged_append_fp4(a["qkv"], c.k_pool, c.v_pool, c.table, c.lengths, a["cos"], a["sin"], a["n_heads"], a["n_kv"],
                             offset=a.get("offset", 0), out=a.get("out"), v_scale=a.get("v_scale", 1.0))

    append(RuntimeError)  # on the CPU
    append(ValueError, qkv=qkv[:, :-128])
    append(ValueError, n_kv=4)
    append(ValueError, offset=-1)
    append(ValueError, v_scale=0.3)
    append(ValueError, out=torch.zeros(2, 12, 64).half())
    append(RuntimeError, qkv=qkv.float())
    append(RuntimeError, cos=cos.bfloat16(), sin=cos.bfloat16())


def test_refuses_a_device_that_is_not_the_current_one(monkeypatch):
    from kernels import _lib, paged_fp4

    def no_entry():
        raise AssertionError("the C entry was reached")

    c = Fp4Case([(1, 20), (1, 5)], spoil=False, device="cpu")
    monkeypatch.setattr(_lib, "_current_device", lambda: 1)
    monkeypatch.setattr(_lib, "lib", no_entry)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    cos = torch.zeros(40, 64)
    pools = (c.k_pool, c.v_pool)
    for call in (lambda: paged_fp4.paged_attention_fp4(c.q, *pools, c.table, c.lengths),
                 lambda: paged_fp4.shared_prefix_attention_fp4(c.q, *pools, c.table[0], 10, c.table, c.lengths),
                 lambda: paged_fp4.paged_append_fp4(torch.zeros(2, 16 * 128).half(), *pools, c.table, c.lengths, cos, cos, 12, 2),
                 lambda: paged_fp4.paged_read_fp4(*pools, c.table, c.lengths)):
        with pytest.raises(RuntimeError, match="current device is cuda:1"):
            call()


def test_c_entries_refuse_without_a_gpu():
    """The C entry points return a status and a message for what they cannot take, before any CUDA call."""
    from kernels import _lib

    h = _lib.lib()

    def attend(entry=h.dk_paged_attention_fp4, **more):
        a = dict(T=2, B=2, nq=12, nkv=2, hd=128, page=16, dtype=0, ldq=1536, pages=4, width=2, starts=0, window=0, sinks=0, prefix=0,
                 k=1.0, v=1.0)
        a.update(more)
        return entry(_lib.PAGED_ATTENTION_FP4_ARGS.pack(
            0, a["ldq"], 0, 0, a["pages"], a["page"], 0, a["prefix"], 0, a["width"], a["width"], 0, a["starts"], a["window"], a["sinks"], 1.0,
            0, a["T"], a["B"], a["nq"], a["nkv"], a["hd"], a["dtype"], 0, 0, 0, a["k"], a["v"]))

    def append(**more):
        a = dict(T=2, B=2, page=16, hd=128, k=1.0)
        a.update(more)
        return h.dk_paged_append_fp4(_lib.PAGED_APPEND_FP4_ARGS.pack(0, 0, 0, 0, 4, a["page"], 0, 2, 2, 0, 0, 0, 0, 1, 64, 10, 0, 0, a["T"],
                                                                     a["B"], 12, 2, a["hd"], 0, 0, a["k"], 1.0))

    def read(**more):
        a = dict(T=2, B=2, page=16, hd=128, nkv=2, dtype=0, pages=4, width=2, starts=0, v=1.0)
        a.update(more)
        return h.dk_paged_read_fp4(_lib.PAGED_READ_FP4_ARGS.pack(0, 0, a["pages"], a["page"], 0, a["width"], a["width"], 0, a["starts"], 1.0,
                                                                 a["v"], 0, 0, a["T"], a["B"], a["nkv"], a["hd"], a["dtype"], 0))

    for entry in (h.dk_paged_attention_fp4, h.dk_shared_prefix_attention_fp4, h.dk_paged_append_fp4, h.dk_paged_read_fp4):
        assert entry(None) == -1
    for entry in (h.dk_paged_attention_fp4, h.dk_shared_prefix_attention_fp4):
        assert attend(entry) == -1 and b"NULL" in h.dk_last_error()
        assert attend(entry, T=3) == -1 and b"one token" in h.dk_last_error()
        assert attend(entry, hd=96) == -3 and attend(entry, page=24) == -3 and attend(entry, nq=13) == -3 and attend(entry, dtype=2) == -3
        assert attend(entry, ldq=8) == -1 and attend(entry, pages=1 << 26) == -1 and attend(entry, width=1 << 27) == -1
        assert attend(entry, T=0, B=0) == attend(entry, T=0, B=3, starts=256) == 0 and attend(entry, T=2, B=0, starts=256) == -1
        for bad in (0.0, 3.0, -2.0, math.inf, math.nan, 2.0 ** 65):
            assert attend(entry, k=bad) == -1 and b"powers of two" in h.dk_last_error()
            assert attend(entry, v=bad) == -1
    assert attend(width=1 << 60) == -1 and attend(window=1 << 31) == -1 and attend(sinks=1 << 40) == -1
    assert append() == -1 and b"NULL" in h.dk_last_error()
    assert append(T=3) == -1 and append(page=20) == -3 and append(hd=96) == -3 and append(k=0.7) == -1 and append(T=0, B=0) == 0
    assert read() == -1 and b"NULL" in h.dk_last_error()
    assert read(T=3) == -1 and b"one row" in h.dk_last_error()
    assert read(page=20) == -3 and read(hd=96) == -3 and read(dtype=2) == -3 and read(v=0.7) == -1 and read(T=2, B=0, starts=256) == -1
    assert read(T=0, B=0) == 0 and read(width=1 << 60) == -1 and read(pages=1 << 40) == -1 and read(nkv=1 << 20) == -1


def test_arguments_are_as_long_as_the_header_says():
    """The packed argument structs have the header's fields, all of 8 bytes."""
    import re
    from pathlib import Path

    from kernels import _lib

    text = (Path(__file__).resolve().parents[1] / "include" / "decodek.h").read_text()

    def fields(name):
        body = re.search(r"typedef struct " + name + r" \{(.*?)\} " + name + ";", text, re.S).group(1)
        n = 0
        for line in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
            if line.strip():
                inner = re.match(r"\s*(dk_paged_\w+_args) \w+$", line)
                n += fields(inner.group(1)) if inner else line.count(",") + 1
        return n

    for name, layout in (("append_fp4", _lib.PAGED_APPEND_FP4_ARGS), ("read_fp4", _lib.PAGED_READ_FP4_ARGS),
                         ("attention_fp4", _lib.PAGED_ATTENTION_FP4_ARGS)):
        assert layout.size == 8 * fields(f"dk_paged_{name}_args")
