"""Edges of the ops over a 4-bit paged cache: roundings on the borders of the format, and calls whose arguments contradict one another."""

import pytest
import torch

from _paged_fp4 import quantise, unpack

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_keys_are_rounded_by_way_of_fp32(dtype):
    """A rotated key is a sum in fp64, rounded to fp32 and from there to the type. Two keys a hair (2^-40) beside the middle between two
    values of the type, one of which is a border between codes: fp32 rounds them to that middle, the type to the border, and the border goes
    to the even code. A single rounding would give the other neighbour, and the other code."""
    from kernels.paged_fp4 import fp4_pages, paged_append_fp4

    half_step = 2.0 ** -10 if dtype is F16 else 2.0 ** -7  # of the type, between 2 and 4
    x, cos, sin = torch.zeros(64, dtype=torch.float64), torch.ones(1, 32, dtype=torch.float64), torch.zeros(1, 32, dtype=torch.float64)
    x[1] = 6  # the group's scale is 1
    for dim, border, side in ((0, 2.5, 1), (2, 3.5, -1)):
        x[dim], x[dim + 32] = 1, 2.0 ** -14
        cos[0, dim], sin[0, dim] = border + side * half_step, -side * 2.0 ** -26
    turned = torch.cat([x[:32] * cos[0] - x[32:] * sin[0], x[32:] * cos[0] + x[:32] * sin[0]])
    assert turned[0] > 2.5 + half_step and turned[2] < 3.5 - half_step
    assert torch.equal(cos, cos.float().double()) and torch.equal(x, x.to(dtype).double())
    rounded = turned.float().to(dtype)
    assert rounded[0] == 2.5 and rounded[2] == 3.5
    k, v = (fp4_pages(1, 1, 16, 64, "cuda").zero_() for _ in range(2))
    qkv = torch.cat([torch.zeros(64), x, torch.zeros(64)]).to(dtype).cuda()[None]
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    paged_append_fp4(qkv, k, v, one[None] - 1, one, cos.float().cuda(), sin.float().cuda(), 1, 1)
    codes, scales = unpack(k.cpu())
    want = quantise(rounded)
    assert torch.equal(codes[0, 0, 0], want[0]) and torch.equal(scales[0, 0, 0], want[1])
    assert codes[0, 0, 0, :3].tolist() == [4, 7, 6]  # 2 and not 3, 6, 4 and not 3


@pytest.mark.gpu
@pytest.mark.parametrize("power", [2.0 ** 64, 2.0 ** -64])
def test_append_and_read_at_the_ends_of_the_powers_range(power):
    """Values around the power, from too small for the smallest scale to too large for the largest."""
    from kernels.paged_fp4 import fp4_pages, paged_append_fp4, paged_read_fp4

    T, hd = 64, 128
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, hd, generator=g, dtype=torch.float64) * torch.logspace(-4, 5, T, dtype=torch.float64)[:, None] * power
    x = x.to(BF16)
    k, v = (fp4_pages(4, 1, 16, hd, "cuda") for _ in range(2))
    table, length = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device="cuda"), torch.tensor([T], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    cos, sin = torch.ones(T, hd // 2, device="cuda"), torch.zeros(T, hd // 2, device="cuda")
    scales = {"k_scale": power, "v_scale": power}
    paged_append_fp4(torch.cat([x, x, x], 1).cuda(), k, v, table, length, cos, sin, 1, 1, starts, **scales)
    want = quantise(x, power)[2]
    for got in paged_read_fp4(k, v, table, length, starts, tokens=T, dtype=BF16, **scales):
        assert torch.equal(got[:, 0].double().cpu(), want)


def test_a_read_whose_rows_contradict_its_outputs_is_refused():
    """`out` and `tokens` both say how many rows there are; one that says otherwise is not dropped silently."""
    from _paged_fp4 import Fp4Case
    from kernels.paged_fp4 import paged_read_fp4

    c = Fp4Case([(3, 20), (2, 5)], spoil=False, device="cpu", one_token=False)
    out = tuple(torch.zeros(5, 2, 128, dtype=F16) for _ in range(2))
    args = (c.k_pool, c.v_pool, c.table, c.lengths, c.starts)
    for tokens in (0, 3, 6):
        with pytest.raises(ValueError, match="tokens"):
            paged_read_fp4(*args, tokens=tokens, out=out)
    for tokens in (None, 5):  # as far as the device
        with pytest.raises(RuntimeError, match="CUDA device"):
            paged_read_fp4(*args, tokens=tokens, out=out)
    for pair in (out[:1], (*out, out[0])):
        with pytest.raises(ValueError, match="out must be two"):
            paged_read_fp4(*args, out=pair)


@pytest.mark.parametrize("fp4", [True, False])
@pytest.mark.parametrize("tokens", [1, 100])
def test_a_call_whose_chunks_pass_64_bits_is_refused(fp4, tokens):
    """2^26 sequences that share a row of 2^26 pages (a table of stride 0), 65535 kv heads: 2^65 chunks are more than 2^30, although
    their number's low 64 bits are less."""
    from kernels import _lib

    h, at, B, nkv, width = _lib.lib(), 1 << 20, 1 << 26, 65535, 1 << 26  # addresses that are looked at for their alignment alone
    args = (at, nkv * 64, at, at, 1, 16, 0, 0, at, 0, width, at, at, 0, 0, 1.0, at, tokens, B, nkv, nkv, 64, 0, at, 0, 0)
    status = (h.dk_paged_attention_fp4(_lib.PAGED_ATTENTION_FP4_ARGS.pack(*args, 1.0, 1.0)) if fp4
              else h.dk_paged_attention(_lib.PAGED_ATTENTION_ARGS.pack(*args)))
    assert status == -3 and b"more than 2^30 chunks" in h.dk_last_error()


def test_workspaces_of_more_positions_than_a_table_can_have_are_refused():
    import ctypes

    from kernels import _lib

    n = ctypes.c_uint64(0)
    for positions, status in ((0, -1), (2 ** 31, -1), (2 ** 63 - 1, -1), (2 ** 31 - 1, 0)):
        assert _lib.lib().dk_paged_attention_fp4_workspace_bytes(1, 1, 12, 2, 128, 0, 1, 0, positions, ctypes.byref(n)) == status
