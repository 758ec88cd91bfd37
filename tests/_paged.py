"""Paged-cache cases for the tests, and the plain 64-bit implementations that the kernels are compared with."""

import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # unit roundoff


class Case:
    """Sequences of `sizes` = [(tokens of the call, positions with them)] in shuffled pages. `spoil`: every page position
    that no sequence owns holds NaN or an infinity, and unused table entries point outside the pool."""

    def __init__(self, sizes, nq=12, nkv=2, hd=128, page=16, dtype=torch.float16, seed=0, one_token=None, spoil=True,
                 prefix=0, device="cuda", wide=1):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.nq, self.nkv, self.hd, self.page, self.dtype = sizes, nq, nkv, hd, page, dtype
        self.T = sum(n for n, _ in sizes)
        need = [-(-max(n, 0) // page) for _, n in sizes]
        extra = -(-prefix // page)
        total = sum(need) + extra + 2
        order = torch.randperm(total, generator=g)
        k = torch.randn(total, nkv, page, hd, generator=g)
        v = torch.randn(total, nkv, page, hd, generator=g)
        used = torch.zeros(total, page, dtype=torch.bool)
        table = torch.full((len(sizes), max(need + [1]) + wide), -7 if spoil else 0, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            for j in range(max(sizes[b][1], 0)):
                used[order[at + j // page], j % page] = True
            at += n
        self.prefix, self.prefix_table = prefix, order[at:at + extra].to(torch.int32)
        for j in range(prefix):
            used[self.prefix_table[j // page].long(), j % page] = True
        if spoil:
            bad = torch.tensor([math.nan, math.inf, -math.inf])
            junk = bad[torch.randint(0, 3, k.shape, generator=g)]
            free = ~used[:, None, :, None]
            k, v = torch.where(free, junk, k), torch.where(free, junk, v)
        self.k, self.v = k.to(device, dtype), v.to(device, dtype)
        self.used = used
        self.table, self.prefix_table = table.to(device), self.prefix_table.to(device)
        self.lengths = torch.tensor([n for _, n in sizes], dtype=torch.int32, device=device)
        starts = torch.tensor([0] + [n for n, _ in sizes]).cumsum(0).to(torch.int32)
        one = all(n == 1 for n, _ in sizes) if one_token is None else one_token
        self.starts = None if one else starts.to(device)
        self.q = torch.randn(self.T, nq, hd, generator=g).to(device, dtype)

    def sequence(self, pool, b):
        """[positions, kv heads, hd] of sequence b (its prefix first) in 64 bits, on the CPU."""
        n = max(self.sizes[b][1], 0)
        j = torch.arange(n)
        own = pool.cpu()[self.table[b].cpu().long()[j // self.page], :, j % self.page]
        i = torch.arange(self.prefix)
        before = pool.cpu()[self.prefix_table.cpu().long()[i // self.page], :, i % self.page]
        return torch.cat([before, own]).double()

    def attention(self, window=0, sinks=0, scale=None):
        """(exact output, tolerance) [T, nq, hd] in 64 bits.

        The tolerance adds up what the kernels round: the output (u |o|), the probabilities to the cache's type before
        the product with v (u sum p |v|; fp16 ones below 2^-14 to a multiple of 2^-24, so 2^-25 each), and the
        scores and exponentials in fp32 (2^-13 of sum p |v| is more than their error: |score| is below 64 here)."""
        scale = self.hd ** -0.5 if scale is None else scale
        u, group = UNIT[self.dtype], self.nq // self.nkv
        out, tol = torch.zeros(self.T, self.nq, self.hd, dtype=torch.float64), torch.zeros(self.T, self.nq, self.hd, dtype=torch.float64)
        t, q = 0, self.q.double().cpu()
        for b, (new, n) in enumerate(self.sizes):
            k, v = self.sequence(self.k, b), self.sequence(self.v, b)
            j = torch.arange(k.shape[0])
            for i in range(new):
                p = self.prefix + n - new + i
                see = j <= p
                if n - new + i < 0 and not self.prefix:
                    see[:] = False
                if window > 0:
                    see &= (j > p - window) | (j < sinks)
                if see.any():
                    ks, vs = k[see].repeat_interleave(group, 1), v[see].repeat_interleave(group, 1)
                    a = torch.softmax(torch.einsum("hd,jhd->hj", q[t], ks) * scale, -1)
                    out[t] = torch.einsum("hj,jhd->hd", a, vs)
                    spread = torch.einsum("hj,jhd->hd", a, vs.abs())
                    tol[t] = u * out[t].abs() + (u + 2.0 ** -13) * spread + see.sum() * 2.0 ** -25 * vs.abs().max()
                t += 1
        return out, tol


def assert_within(got, exact, tol):
    off = (got.double().cpu() - exact).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert torch.isfinite(got.float()).all()
    assert worst <= 0, f"{worst:.3g} over the tolerance; largest error {off.max().item():.3g}"
