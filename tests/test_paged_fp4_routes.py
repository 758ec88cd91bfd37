"""Attention over a 4-bit paged cache on each of its ways: which kernels take a call depends on its tokens, its sequences and the width of
its page table. Each test says which ones its calls have to take, and shows that they do, so that it goes on testing them."""

import pytest
import torch

from _paged import UNIT, assert_within
from _paged_fp4 import Fp4Case
from _routes import kernels_of
from test_paged_fp4 import _attend, _attend_in

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("sizes,wide,route", [
    ([(1, 700), (1, 31)], 1, "one token"),
    ([(3, 300), (2, 200)], 1, "rows"),
    ([(90, 300), (2, 90)], 1 << 16, "split"),
    ([(300, 420)], 1, "copied"),
])
def test_bf16_calls_keep_p_in_fp16(sizes, wide, route, hd, tmp_path):
    """Whichever kernels a bf16 call takes, p has fp16's 11 bits in the product with v: Case.attention's terms with that
    roundoff for the probabilities, and bf16's for the output alone."""
    c = Fp4Case(sizes, nq=12, nkv=2, hd=hd, dtype=BF16, seed=6, one_token=route == "one token", wide=wide)
    window, sinks = 9, 1  # (few positions, so that what one probability is off by is not averaged away)
    assert kernels_of(lambda: _attend(c, window=window, sinks=sinks), tmp_path) & {"rows", "fp4_rows", "fp4_copy", "tiles", "tiles_codes"} == {
        "one token": {"fp4_rows"}, "rows": {"fp4_rows"}, "split": {"fp4_rows", "tiles_codes"}, "copied": {"fp4_copy", "tiles"}}[route]
    exact, _ = c.attention(window, sinks)
    c.dtype = F16
    _, tol = c.attention(window, sinks)  # fp16's roundoff in every term: the output's is exchanged for bf16's
    assert_within(_attend(c, window=window, sinks=sinks), exact, tol + (2.0 ** -8 - 2.0 ** -11) * exact.abs())


# Ragged calls on each of their ways: sequences, query and kv heads, spare columns of the page table, kernels. Calls of little work go to
# the rows kernel, others are split by their sequences' tokens (`limit` of them at most on the rows kernel) or, with 256 tokens a
# sequence and more, taken by the 256-row tiles, which read a 16-bit copy where a sequence has three tiles and the copy fits.
ROUTES = {
    "rows": ([(9, 200), (4, 140), (5, 60)], 6, 2, 1, {"plan", "fp4_rows"}),
    "split": ([(60, 300), (9, 90), (4, 200)], 6, 2, 1 << 16, {"plan_both", "fp4_rows", "tiles_codes"}),
    "tiles": ([(300, 420), (230, 260)], 6, 2, 1 << 16, {"plan", "tiles_codes"}),
    "copied": ([(300, 420), (230, 260)], 6, 2, 1, {"fp4_copy", "tiles"}),
    "copied, split": ([(200, 260), (3, 77), (90, 180), (60, 400)], 16, 1, 200, {"fp4_copy", "fp4_rows", "tiles"}),
}


def _case(route, page=16, **more):
    sizes, nq, nkv, wide, _ = ROUTES[route]
    return Fp4Case(sizes, nq=nq, nkv=nkv, page=page, one_token=False, wide=wide, **more)


def _takes(route, c, tmp_path, **more):
    """Asserts that the call goes the way it is meant to go."""
    names = kernels_of(lambda: _attend(c, **more), tmp_path)
    assert {n for n in names if not n.startswith("join")} == ROUTES[route][4], names


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd,page", [(F16, 128, 16), (BF16, 128, 256), (BF16, 64, 32)])
@pytest.mark.parametrize("route", ROUTES)
def test_masks(route, dtype, hd, page, tmp_path):
    """Windows and sinks that end in their page, at its end, before the window's first page and beyond, in workspaces that hold
    something."""
    c = _case(route, page, dtype=dtype, hd=hd, seed=2, k_scale=0.5, v_scale=2.0)
    for window, sinks in ((0, 0), (100, 0), (100, 17), (33, 64), (1, 3), (200, 300)):
        out = _attend_in(c, 1, window, sinks)
        assert_within(out, *c.attention(window, sinks))
        assert torch.equal(out, _attend_in(c, -1, window, sinks))
        _takes(route, c, tmp_path, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("pool", ["k_pool", "v_pool"])
@pytest.mark.parametrize("route", ROUTES)
def test_a_nan_reaches_the_rows_that_see_it(route, pool, dtype, hd, tmp_path):
    """A NaN scale at position 3 of the first sequence makes all of its rows' results of the last kv head NaN, and nothing else."""
    c = _case(route, dtype=dtype, hd=hd, seed=12)
    getattr(c, pool)[c.table[0, 0].long(), c.nkv - 1].view(-1)[16 * hd // 2 + 3 * hd // 16] = 0x7f
    out, n, group = _attend(c), c.sizes[0][0], c.nq // c.nkv
    bad = out[:n, c.nq - group:].isnan()
    assert bad.all() if pool == "k_pool" else bad[..., :16].all() and not bad[..., 16:].any()
    assert out[:n, :c.nq - group].isfinite().all() and out[n:].isfinite().all()
    _takes(route, c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("route", ROUTES)
def test_visible_positions_without_a_page_are_zeros_and_reported(route, window, dtype, hd, tmp_path):
    from kernels import _lib

    c = _case(route, dtype=dtype, hd=hd, seed=13, spoil=False)
    _lib.clear_device_error()
    assert_within(_attend(c, window=window, sinks=2), *c.attention(window, 2))
    assert _lib.device_error() == 0
    own, at = c.table, (c.sizes[0][1] - 10) // c.page
    after = c.table.clone()
    after[0, -(-c.sizes[0][1] // c.page):] = 1 << 30  # behind the last position
    c.table = after
    assert_within(_attend(c, window=window, sinks=2), *c.attention(window, 2))
    assert _lib.device_error() == 0
    lost = own[0, at].long().item()
    c.table = own
    c.k[lost], c.v[lost] = 0, 0
    want = c.attention(window, 2)
    for entry in (-1, c.k_pool.shape[0], 2 ** 31 - 1):
        c.table = own.clone()
        c.table[0, at] = entry
        out = _attend_in(c, -1, window, 2)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        assert_within(out, *want)
    _takes(route, c, tmp_path, window=window, sinks=2)
    _lib.clear_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("route", ROUTES)
def test_freed_pages_are_left_alone(route, dtype, hd, tmp_path):
    """Pages between the sinks and the window may be gone: their table entries point nowhere, their bytes are NaN."""
    from kernels import _lib

    c = _case(route, dtype=dtype, hd=hd, seed=3)
    window, sinks = 50, 4
    want = c.attention(window, sinks)
    for b, (new, n) in enumerate(c.sizes):
        first, last = 1, (n - new + 1 - window) // c.page
        for i in range(first, last):
            gone = c.table[b, i].long().item()
            c.k_pool[gone], c.v_pool[gone] = 0x7f, 0x7f
        if last > first:
            c.table[b, first:last] = torch.tensor([-1, 1 << 30]).repeat(last)[:last - first].int()
    _lib.clear_device_error()
    assert_within(_attend_in(c, -1, window, sinks), *want)
    assert _lib.device_error() == 0
    _takes(route, c, tmp_path, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("size", [2.0 ** -8, 60.0])
@pytest.mark.parametrize("route", ROUTES)
def test_queries_of_any_size(route, size, dtype, tmp_path):
    """Scores far apart and all alike, heads that differ by orders of magnitude, one of zeros; uneven rows of a bf16 call are those
    whose power of two matters. Beside Case.attention's terms: a score is a sum of 128 exact products in eight steps of fp32, each off by less than
    2^-23 of sum |q| |k|, so by up to 2^-20 of that, and so are the weights, above and below the division."""
    c = _case(route, dtype=dtype, seed=5)
    c.q *= size
    c.q[0, 0] *= 2.0 ** -12
    c.q[0, 1] = 0
    c.q[-1, 0, ::3] *= 2.0 ** -9
    exact, tol = c.attention()
    group, t = c.nq // c.nkv, 0
    for b, (new, n) in enumerate(c.sizes):
        k, v = c.sequence(c.k, b).abs().repeat_interleave(group, 1), c.sequence(c.v, b).abs().amax(0).repeat_interleave(group, 0)
        for i in range(new):
            most = torch.einsum("hd,jhd->hj", c.q[t].double().cpu().abs(), k[:n - new + i + 1]).amax(-1) * c.hd ** -0.5
            tol[t] += (2.0 ** -19 * most)[:, None] * v
            t += 1
    assert_within(_attend(c), exact, tol)
    _takes(route, c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.15, 1e-60])
@pytest.mark.parametrize("route", ROUTES)
def test_scales_of_any_sign(route, scale, dtype, hd, tmp_path):
    """Zero weighs the visible positions alike, a negative scale the smallest products most; masked positions stay out of it."""
    c = _case(route, dtype=dtype, hd=hd, seed=10)
    for window, sinks in ((0, 0), (50, 3)):
        assert_within(_attend(c, window=window, sinks=sinks, scale=scale), *c.attention(window, sinks, scale=scale))
    _takes(route, c, tmp_path, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** 64, 2.0 ** -64), (2.0 ** -64, 2.0 ** 64)])
@pytest.mark.parametrize("route", ROUTES)
def test_powers_at_the_ends_of_their_range(route, k_scale, v_scale, tmp_path):
    """Queries as small (as large) as the keys' power is large (small): all of it is shifts of exponents."""
    c = _case(route, dtype=BF16, seed=17, k_scale=k_scale, v_scale=v_scale)
    for window, sinks in ((0, 0), (40, 3)):
        assert_within(_attend(c, window=window, sinks=sinks), *c.attention(window, sinks))
    _takes(route, c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("before,after", [(2, 0), (0, 5), (3, 7)])
@pytest.mark.parametrize("route", ROUTES)
def test_rows_outside_starts_are_zeros(route, before, after, dtype, hd, tmp_path):
    c = _case(route, dtype=dtype, hd=hd, seed=14)
    exact, tol = c.attention()
    live = slice(before, before + c.T)
    q = torch.randn(before + c.T + after, c.nq, c.hd, device="cuda").to(dtype)
    q[live] = c.q
    c.q, c.starts = q, c.starts + before
    out = torch.full_like(c.q, torch.nan)
    _attend(c, out=out)
    assert_within(out[live], exact, tol)
    assert not out[:before].any() and not out[before + c.T:].any()
    _takes(route, c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("before,after", [(0, 700), (3, 5)])
def test_rows_outside_starts_beside_tiles_without_work(before, after, dtype, hd, tmp_path):
    """The call might have prompts, but its sequences have few tokens: the tiles' launch writes nothing but the zeros."""
    c = Fp4Case([(3, 20), (2, 200), (4, 0)], hd=hd, dtype=dtype, one_token=False, wide=1 << 16, seed=15)
    exact, tol = c.attention()
    own = c.q
    c.q = torch.randn(before + c.T + after, c.nq, c.hd, device="cuda").to(dtype)
    c.q[before:before + c.T], c.starts = own, c.starts + before
    out = torch.full_like(c.q, torch.nan)
    _attend(c, out=out)
    assert_within(out[before:before + c.T], exact, tol)
    assert not out[:before].any() and not out[before + c.T:].any()
    _takes("split", c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("sinks", [0, 3, 40])
@pytest.mark.parametrize("route", ROUTES)
def test_windows_wholly_past_the_table_leave_the_sinks(route, sinks, tmp_path):
    """A length past the table is reported; what counts is what the table has of the window (nothing) and the sinks."""
    from kernels import _lib

    c = _case(route, seed=16)
    own, new, window = c.lengths, c.sizes[0][0], 20
    exact, tol = c.attention(window, sinks)
    k, v, group = c.sequence(c.k, 0)[:sinks], c.sequence(c.v, 0)[:sinks], c.nq // c.nkv
    for t in range(new):  # of the first sequence: over the positions 0..sinks - 1, with the tolerance of Case.attention
        exact[t], tol[t] = 0, 0
        if sinks:
            a = torch.softmax(torch.einsum("hd,jhd->hj", c.q[t].double().cpu(), k.repeat_interleave(group, 1)) * c.hd ** -0.5, -1)
            vs, u = v.repeat_interleave(group, 1), UNIT[c.dtype]
            exact[t] = torch.einsum("hj,jhd->hd", a, vs)
            tol[t] = u * exact[t].abs() + (u + 2.0 ** -13) * torch.einsum("hj,jhd->hd", a, vs.abs()) + sinks * 2.0 ** -25 * vs.abs().max()
    for length in (c.table.shape[1] * c.page + new + window + 7, 2 ** 31 - 1):
        c.lengths = own.clone()
        c.lengths[0] = length
        _lib.clear_device_error()
        out = _attend(c, window=window, sinks=sinks)
        assert _lib.device_error() == 3  # DK_DEVERR_BAD_POSITION
        _lib.clear_device_error()
        assert_within(out, exact, tol)
    c.lengths = own
    _takes(route, c, tmp_path, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("route", ROUTES)
def test_strides_stream_and_graph(route, dtype, tmp_path):
    """Query rows inside a wider tensor, a table that is part of a wider one, a side stream, a captured call whose inputs then change."""
    c = _case(route, dtype=dtype, seed=4, k_scale=0.5, v_scale=4.0)
    want = c.attention(60, 5, scale=0.2)
    wide = torch.zeros(c.T, c.nq + 5, c.hd, dtype=dtype, device="cuda")
    wide[:, :c.nq] = c.q
    table = torch.full((len(c.sizes), c.table.shape[1] + 8), -1, dtype=torch.int32, device="cuda")
    table[:, :-8] = c.table
    c.q, c.table = wide[:, :c.nq], table[:, :-8]
    more = dict(window=60, sinks=5, scale=0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = _attend(c, **more)
    torch.cuda.current_stream().wait_stream(side)
    assert_within(out, *want)
    graph, kept = torch.cuda.CUDAGraph(), torch.empty_like(out)
    with torch.cuda.graph(graph):
        _attend(c, out=kept, **more)
    graph.replay()
    assert torch.equal(kept, out)
    # the same graph serves other lengths and tokens
    c.lengths.sub_(torch.tensor([min(7, n - 1) for _, n in c.sizes], dtype=torch.int32, device="cuda"))
    c.q.mul_(0.5)
    graph.replay()
    c.sizes = [(new, n - min(7, n - 1)) for new, n in c.sizes]
    assert_within(kept, *c.attention(60, 5, scale=0.2))
    _takes(route, c, tmp_path, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("sizes,by_unit", [
    ([(2, 40)] * 70, False),  # no tiles, as many units of them as CTAs may come
    ([(1, 900), (2, 40)] * 40, False),
    ([(2, 40)] * 69 + [(60, 300)], False),
    ([(3, 40)] * 9, True),  # fewer units
    ([(30, 900), (2, 40), (24, 30), (25, 30)], True),
])
def test_launches_without_work_leave_no_records_for_the_join(sizes, by_unit, dtype, hd, tmp_path):
    """The join of a split call reads what the tiles' launch left for each CTA, or with fewer units than CTAs the plan: of a
    launch without work too, whatever the workspace held."""
    c = Fp4Case(sizes, nq=8, nkv=4, hd=hd, page=16, dtype=dtype, seed=11, one_token=False, wide=1 << 16)
    tile = 2 * 128 // 2  # tokens of two heads
    assert ((c.T // tile + len(sizes)) * 4 < torch.cuda.get_device_properties(0).multi_processor_count) == by_unit
    out = _attend_in(c, 1)
    assert_within(out, *c.attention())
    assert torch.equal(out, _attend_in(c, 0)) and torch.equal(out, _attend_in(c, -1))
    _takes("split", c, tmp_path)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,dtype", [(64, F16), (128, BF16)])
def test_long_rings_of_copied_prompts_give_the_right_rows(hd, dtype, tmp_path):
    """Many more chunks than a ring has slots, every row compared."""
    c = Fp4Case([(900, 2500), (300, 1500)], nq=6, nkv=2, hd=hd, page=32, seed=8, spoil=False, dtype=dtype)
    assert_within(_attend(c), *c.attention())
    _takes("copied", c, tmp_path)


def test_split_calls_count_each_launch_by_what_it_takes():
    """Of a call that is split by its sequences' tokens, the launch for the short ones has three tiles a sequence at most, however many
    tokens the others bring: 2048 sequences of 195 tokens on average, 64 heads over 8, tables of 131072 positions are no more work than
    the library takes (as far as the workspace, of which there is none), 65536 such sequences are."""
    from kernels import _lib

    h = _lib.lib()

    def attend(T, B):
        at, width = 1 << 20, 131072 // 64  # addresses that are looked at for their alignment alone
        return h.dk_paged_attention_fp4(_lib.PAGED_ATTENTION_FP4_ARGS.pack(
            at, 64 * 128, at, at, 1 << 20, 64, 0, 0, at, width, width, at, at, 0, 0, 1.0, at, T, B, 64, 8, 128, 0, at, 0, 0, 1.0, 1.0))

    assert attend(400_000, 2048) == -1 and b"the workspace has 0 bytes" in h.dk_last_error()
    assert attend(12_800_000, 65536) == -3 and b"chunks" in h.dk_last_error()
