"""4-bit paged-cache cases for the tests, and the format's plain 64-bit implementation."""

import torch

from _paged import Case

NUMBERS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)  # E2M1
SCALES = torch.tensor([(1 + b % 8 / 8) * 2.0 ** (b // 8 - 7) if b >= 8 else b * 2.0 ** -9 for b in range(127)],
                      dtype=torch.float64)  # E4M3 without a sign; 127 is NaN


def nearest(x, values):
    """Index of the value nearest to x >= 0 (none larger than the last), ties to the even index."""
    x = x.clamp(max=values[-1].item())
    even, i = (x[..., None] - values[0::2]).abs().min(-1)
    odd, j = (x[..., None] - values[1::2]).abs().min(-1)
    return torch.where(odd < even, 2 * j + 1, 2 * i)


def quantise(x, power=1.0):
    """x [..., dim] (values of a 16-bit type) -> codes 0..15 [..., dim], scale bytes [..., dim / 16], values [..., dim] in 64 bits."""
    x = x.double().unflatten(-1, (-1, 16))
    top = x.abs().amax(-1)
    scale = torch.where(top.isnan(), 127, nearest(torch.nan_to_num(top / 6 / power, nan=0.0, posinf=1e9), SCALES))
    unit = torch.where(scale == 127, torch.nan, SCALES[scale.clamp(max=126)])[..., None]
    ratio = torch.where(unit > 0, x.abs() / power / unit.clamp(min=2.0 ** -20), torch.zeros_like(x))
    size = nearest(torch.nan_to_num(ratio, nan=0.0, posinf=1e9), NUMBERS)
    sign = torch.signbit(x)
    values = NUMBERS[size] * unit * power * torch.where(sign, -1.0, 1.0)
    return (size + 8 * sign).flatten(-2), scale, values.flatten(-2)


def pack(codes, scales):
    """codes [pages, kv, page, dim], scale bytes [pages, kv, page, dim / 16] -> a pool."""
    n, kv, page, dim = codes.shape
    bytes_of = codes[..., 0::2] + 16 * codes[..., 1::2]
    flat = torch.cat([bytes_of.flatten(2), scales.flatten(2)], -1)
    return flat.to(torch.uint8).view(n, kv, page, dim * 9 // 16)


def unpack(pool):
    """A pool's codes [pages, kv, page, dim] and scale bytes [pages, kv, page, dim / 16]."""
    n, kv, page, row = pool.shape
    dim = row * 16 // 9
    flat = pool.reshape(n, kv, page * row).long()
    codes = flat[..., :page * dim // 2].view(n, kv, page, dim // 2)
    return torch.stack([codes % 16, codes // 16], -1).flatten(-2), flat[..., page * dim // 2:].view(n, kv, page, dim // 16)


class Fp4Case(Case):
    """A Case whose cache is held in 4 bits: k_pool and v_pool are the pools, k and v what they stand for (64 bits, on the CPU).
    `spoil`: positions of no sequence hold NaN scales and saturated codes. Values are of a size that suits the powers."""

    def __init__(self, *args, k_scale=1.0, v_scale=1.0, device="cuda", **more):
        super().__init__(*args, device="cpu", **more)
        self.k_scale, self.v_scale = k_scale, v_scale
        pools = []
        for name, power in (("k", k_scale), ("v", v_scale)):
            codes, scales, values = quantise(getattr(self, name).double() * power, power)
            pools.append(pack(codes, scales).to(device))
            setattr(self, name, values)
        self.k_pool, self.v_pool = pools
        for name in ("table", "prefix_table", "lengths", "starts", "q"):
            x = getattr(self, name)
            setattr(self, name, x if x is None else x.to(device))
        self.q = (self.q.double() / k_scale).to(self.dtype)
        self.scales = {"k_scale": k_scale, "v_scale": v_scale}
