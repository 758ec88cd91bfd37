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
