"""Attention over a 4-bit paged cache on each of its ways: which kernels take a call depends on its tokens, its sequences and the width of
its page table. Each test says which ones its calls have to take, and shows that they do, so that it goes on testing them."""

import pytest
import torch

from _paged import assert_within
from _paged_fp4 import Fp4Case
from _routes import kernels_of
from test_paged_fp4 import _attend

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
