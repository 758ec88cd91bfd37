"""Token log probabilities (kernels.logprobs.token_logprobs, C-ABI dk_token_logprobs) against a plain 64-bit
implementation: values, entropy, and the top alternatives with their ties."""

import math

import pytest
import torch

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _exact(x, targets, top):
    x = x.double().cpu()
    logp = torch.log_softmax(x, -1)
    lp = torch.where(targets.cpu() >= 0, logp.gather(1, targets.cpu().clamp(min=0)[:, None])[:, 0], torch.zeros(len(x)).double())
    entropy = -torch.where(logp > -math.inf, logp.exp() * logp, torch.zeros_like(logp)).sum(-1)
    value, index = torch.sort(logp, dim=-1, descending=True, stable=True)
    return lp, entropy, value[:, :top], index[:, :top]


def _check(x, targets, top):
    from kernels.logprobs import token_logprobs

    lp, entropy, value, index = (t.cpu() for t in token_logprobs(x, targets, top))
    want = _exact(x, targets, top)
    V = x.shape[1]
    # A thread adds up at most V / 512 + 32 terms (short rows: one tile), each with a relative error below 2^-21 (the
    # exponential and its rounded argument), and a tree joins the threads; then roundings of the result's size.
    eps = (V / 512 + 72) * 2.0 ** -24 + 2.0 ** -21
    assert ((lp - want[0]).abs() <= eps + want[0].abs() * 2.0 ** -22).all()
    assert ((entropy - want[1]).abs() <= eps * (2 + 2 * want[1])).all()
    assert torch.equal(index, want[3])
    fin = want[2] > -math.inf
    assert ((value - want[2]).abs()[fin] <= eps + want[2].abs()[fin] * 2.0 ** -22).all()
    assert torch.equal(value[~fin].double(), want[2][~fin])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,top", [
    (1, 1, 1), (2, 7, 7), (1, 151936, 5), (3, 152064, 20), (5, 1003, 32), (300, 517, 3), (2, 32001, 0), (40, 16385, 16),
    (1, 65537, 17), (150, 20011, 8),
])
def test_logprobs(M, V, top, dtype):
    g = torch.Generator().manual_seed(M * V + top)
    x = (torch.randn(M, V, generator=g) * 3).to(dtype).cuda()
    targets = torch.randint(0, V, (M,), generator=g).cuda()
    targets[0] = -1 if M > 2 else targets[0]
    _check(x, targets, top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,V", [(20, 70001), (60, 70001), (100, 66001), (200, 66001), (400, 9001), (700, 9001)])
def test_rows_over_the_sms(M, V, dtype):
    """Rows split over four CTAs, over two on one SM or on several, whole rows with and without room to spare on the SMs."""
    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, V, generator=g) * 2).to(dtype).cuda()
    _check(x, torch.randint(0, V, (M,), generator=g).cuda(), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_ties_masks_and_orders(dtype):
    """Equal logits, rising and falling rows, all but a few tokens forbidden (-inf or the type's lowest value)."""
    V, top = 40000, 20
    rows = [torch.zeros(V), torch.arange(V) / 4096, -torch.arange(V) / 4096, torch.full((V,), -math.inf),
            torch.full((V,), torch.finfo(dtype).min), (torch.arange(V) % 7).float(), torch.full((V,), -0.0)]
    rows[3][[5, 17, 39999]] = torch.tensor([1.0, -2.0, 1.0])
    rows[4][[39998, 3]] = torch.tensor([0.5, 0.25])
    rows[6][::3] = 0.0
    x = torch.stack(rows).to(dtype).cuda()
    targets = torch.tensor([V - 1, 0, 1, 17, 3, 6, 2]).cuda()
    _check(x, targets, top)
    for row in range(len(rows)):  # a row alone is split over several CTAs
        _check(x[row:row + 1], targets[row:row + 1], top)


@pytest.mark.gpu
def test_strided_and_unaligned_rows():
    x = torch.randn(9, 5001, device="cuda", dtype=torch.bfloat16)
    targets = torch.arange(9, device="cuda")
    for lo in (0, 1, 3, 8):
        _check(x[:, lo:lo + 4990], targets, 6)
    y = torch.randn(3, 1001, device="cuda")
    _check(y[:, 1:], targets[:3], 32)


@pytest.mark.gpu
def test_nothing_allowed_nan_and_infinity():
    from kernels import _lib
    from kernels.logprobs import token_logprobs

    x = torch.randn(4, 3000, device="cuda", dtype=torch.float16)
    x[0] = -math.inf
    x[1, 100] = math.nan
    x[2, 200] = math.inf
    _lib.clear_device_error()
    lp, entropy, value, index = token_logprobs(x, torch.tensor([1, 2, 3, 3000], device="cuda"), 3)
    assert _lib.device_error() == 6  # DK_DEVERR_BAD_TOKEN: the last row's target
    _lib.clear_device_error()
    assert lp[:3].isnan().all() or (lp[2] == -math.inf and lp[:2].isnan().all())
    assert lp[3].isnan() and entropy[:3].isnan().all() and entropy[3].isfinite()
    assert index[0].tolist() == [0, 1, 2] and index[1, 0] == 100 and index[2, 0] == 200


@pytest.mark.gpu
def test_empty_and_captured():
    from kernels.logprobs import token_logprobs

    lp, entropy, value, index = token_logprobs(torch.zeros(0, 50, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), 4)
    assert lp.shape == entropy.shape == (0,) and value.shape == index.shape == (0, 4)
    x, t = torch.randn(2, 9000, device="cuda"), torch.tensor([1, 2], device="cuda")
    want = token_logprobs(x, t, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, t, 5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_without_a_gpu():
    from kernels import _lib
    from kernels.logprobs import token_logprobs

    x, t = torch.zeros(2, 50), torch.zeros(2, dtype=torch.long)
    for error, a in [(RuntimeError, (x, t)), (ValueError, (x[0], t)), (ValueError, (x, t[:1])), (ValueError, (x, t, 33)),
                     (ValueError, (x, t, -1)), (ValueError, (x[:, :4], t, 5)), (ValueError, (x.T, t)),
                     (ValueError, (x[:1].expand(2, 50), t)), (RuntimeError, (x.double(), t)), (RuntimeError, (x, t.int()))]:
        with pytest.raises(error):
            token_logprobs(*a)
    h = _lib.lib()
    assert h.dk_token_logprobs(None, 50, 0, None, 2, 50, 0, None, None, None, None, None) == -1
    assert h.dk_token_logprobs(None, 49, 0, None, 2, 50, 0, None, None, None, None, None) == -1
    assert h.dk_token_logprobs(None, 50, 0, None, 2, 50, 33, None, None, None, None, None) == -3
    assert h.dk_token_logprobs(None, 50, 7, None, 2, 50, 0, None, None, None, None, None) == -3


def _shared_accesses(warps, rounds, inside):
    """What the warps of logprobs.cu do with the groups' maxima: [(barriers passed, warp, 'r' or 'w', group)]. Every round a warp
    writes its 8 groups, waits, reads them for the threshold (the first two warps), waits; in the first one all warps
    read the largest too, before the second barrier (`inside`) or after it."""
    got = []
    for w in range(warps):
        at = 0
        for i in range(rounds):
            got += [(at, w, "w", 8 * w + g) for g in range(8)]
            at += 1
            if w < 2 or (inside and i == 0):
                got += [(at, w, "r", g) for g in range(8 * warps)]
            at += 1
            if not inside and i == 0:
                got += [(at, w, "r", g) for g in range(8 * warps)]
    return got


def _races(accesses):
    wrote = {}
    for at, w, kind, g in accesses:
        if kind == "w":
            wrote.setdefault((at, g), set()).add(w)
    return [(at, w, g) for at, w, kind, g in accesses if kind == "r" and wrote.get((at, g), set()) - {w}]


@pytest.mark.parametrize("rounds", [1, 2, 3])
def test_threshold_rounds_do_not_race(rounds):
    """No warp reads a group's maximum between the same barriers as another warp writes it; the same reads after the second
    barrier would, from two rounds on."""
    assert not _races(_shared_accesses(8, rounds, inside=True))
    assert bool(_races(_shared_accesses(8, rounds, inside=False))) == (rounds > 1)


@pytest.mark.gpu
@pytest.mark.parametrize("M,V", [(1, 151936), (300, 20011), (600, 70001)])
def test_calls_repeat_bit_for_bit(M, V):
    """Logits that rise along the row, so that the maxima of later rounds differ from the first's: call after call gives the
    same bits."""
    from kernels.logprobs import token_logprobs

    g = torch.Generator().manual_seed(M)
    x = (torch.randn(M, V, generator=g) + torch.arange(V) * (30 / V)).half().cuda()
    targets = torch.randint(0, V, (M,), generator=g).cuda()
    want = token_logprobs(x, targets, 5)
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for _ in range(50):
        for a, b in zip(token_logprobs(x, targets, 5), want):
            same &= (a == b).all()
    assert same.item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,top", [(1, 0), (3, 0), (3, 3), (7, 2), (20, 0), (40000, 0), (40000, 5)])
def test_rows_of_the_lowest_value(V, top, dtype):
    """Rows of nothing but the type's lowest value (a mask added to all tokens), of that and -inf, of that and one ordinary
    logit: short rows without a whole vector, ends outside whole vectors, and rows of many tiles."""
    low = torch.finfo(dtype).min
    rows = torch.full((3, V + 1), low)
    rows[1, 2::3] = -math.inf
    rows[2, 1] = 0.5
    x = rows.to(dtype).cuda()
    for view in (x[:, :V], x[:, 1:]):  # the second one begins off a vector's boundary
        for target in (0, V - 1):
            _check(view, torch.where(view[:, target] == -math.inf, -1, target), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,at", [(3000, 200), (3, 2), (40001, 40000), (40001, 0), (160001, 30000)])
def test_infinity_and_nan_give_nan(V, at, dtype):
    """A row with +inf or NaN anywhere has NaN log probabilities, of its finite tokens and of the infinite one, and entropy."""
    from kernels.logprobs import token_logprobs

    for bad in (math.inf, math.nan):
        x = torch.randn(2, V + 1, device="cuda").to(dtype)
        x[:, at] = bad
        for view in (x[:, :V], x[:1, :V]):
            for target in (at, (at + 1) % V):
                for top in (0, 2):
                    lp, entropy, value, index = token_logprobs(view, torch.full((len(view),), target, device="cuda"), top)
                    assert lp.isnan().all() and entropy.isnan().all() and value.isnan().all()
                    assert (index[:, :1] == at).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_peaked_rows(dtype):
    """One logit far above the others anywhere in the row, as of a sure token: its log probability and the row's entropy are
    next to zero and come out so, on the right side of zero.

    Relative to the maximum its own term is 1 without an error. The others are below 2^-31 each, below 2^-24 for one thread, and below
    2^-20 in all, with a relative error below 2^-15 (their exponents reach 60, and up to V / 512 + 72 roundings). Adding them to 1 loses
    at most a thread's and rounds at most 22 times (the threads' pairs, two trees of 5 steps, 7 other CTAs, ln s), 2^-24 each."""
    from kernels.logprobs import token_logprobs

    V, M = 60000, 64
    g = torch.Generator().manual_seed(20)
    x = torch.randn(M, V, generator=g).clamp(-4, 4)
    at = torch.randint(0, V, (M,), generator=g)
    x[torch.arange(M), at] = 26 + 12 * torch.rand(M, generator=g)
    x, at = x.to(dtype).cuda(), at.cuda()
    for rows in (slice(0, M), slice(0, 1), slice(1, 2)):
        lp, entropy, value, index = (t.cpu() for t in token_logprobs(x[rows], at[rows], 2))
        want = _exact(x[rows], at[rows], 2)
        eps = 23 * 2.0 ** -24
        assert ((lp - want[0]).abs() <= eps + 2.0 ** -15 * want[0].abs()).all() and (lp <= 0).all()
        assert ((entropy - want[1]).abs() <= eps + 2.0 ** -15 * want[1]).all() and (entropy >= 0).all()
        assert torch.equal(index, want[3])
