"""Workloads of the operators around a paged cache held in 4 bits, for timing and for comparing outputs.

A batch server whose contexts no longer fit in 16 bits keeps keys and values as E2M1 numbers (4 bits: a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6) with an E4M3 scale for every 16 dims of a position, and one power of two for a whole pool:
4.5 bits a value. Four operators:

* `append`    rotate q and k by their positions, quantise k and v and write them into the pages, and read the call's own
              positions back;
* `read`      read positions of the cache back, as 16-bit values;
* `attention` attention over the pages, causal, optionally limited to a sliding window plus a few first tokens that stay
              visible; one token per sequence (decode), a few (checking drafted tokens) or ragged rows of them (prompts);
* `prefix`    attention of a batch whose sequences share a long prefix, read once for all of them.

`run` computes them in plain torch, or with `own = True` by the `kernels` package. Head layouts are those of
kernels/config.py (12 query / 2 kv heads and 28 / 4, head_dim 128) and their tensor-parallel shards.

A (page, kv head) of a pool [pages, kv heads, page size, 9/16 head_dim] of bytes holds first the codes, head_dim / 2 bytes a
position (dim 2 i in the low half of byte i), then the scales, head_dim / 16 bytes a position.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "llm-decode-kernels_b200")
_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    heads15 = {"heads": 12, "kv": 2, "dim": 128}
    heads7 = {"heads": 28, "kv": 4, "dim": 128}
    scales = {"k_exp": -2, "v_exp": -4}  # pools whose values come to a few tens (keys with a bias) and below one
    return [
        # one decode step of a batch server: one new token for each of 64 sequences: latency
        {"name": "append decode 64", "op": "append", **heads7, "type": "float16", "page": 64, "batch": 64,
         "tokens": 1, "context": 2048, **scales, "mix": 1},
        # the prompts of a batch, ragged, appended in one call (the second half of each prompt: chunked prefill): bandwidth
        {"name": "append prompts", "op": "append", **heads7, "type": "bfloat16", "page": 16, "batch": 8,
         "tokens": 2048, "context": 4096, **scales, "mix": 2},
        # one short conversation handed to a 16-bit cache: latency
        {"name": "read 1x525", "op": "read", **heads15, "type": "float16", "page": 16, "batch": 1, "tokens": 525,
         "context": 525, **scales, "mix": 3},
        # conversations moved out of the 4-bit cache, whole: bandwidth
        {"name": "read 16x8192", "op": "read", **heads7, "type": "bfloat16", "page": 64, "batch": 16, "tokens": 8192,
         "context": 8192, **scales, "mix": 4},
        # interactive decode of one sequence at the benchmark's prompt length: latency
        {"name": "attention decode 1x640", "op": "attention", **heads15, "type": "float16", "page": 16, "batch": 1,
         "tokens": 1, "context": 640, "window": 0, "sinks": 0, **scales, "mix": 5},
        # decode of a full batch over ragged contexts: bandwidth
        {"name": "attention decode 64x8192", "op": "attention", **heads7, "type": "bfloat16", "page": 64, "batch": 64,
         "tokens": 1, "context": 8192, "window": 0, "sinks": 0, **scales, "mix": 6},
        # long conversations decoded through a window with sink tokens; pages outside it are already freed
        {"name": "attention decode window", "op": "attention", **heads15, "type": "float16", "page": 32, "batch": 48,
         "tokens": 1, "context": 32768, "window": 1024, "sinks": 4, **scales, "mix": 7},
        # drafted tokens of a batch checked in one call: up to five rows behind each context
        {"name": "attention drafts 32x4096", "op": "attention", **heads7, "type": "bfloat16", "page": 32, "batch": 32,
         "tokens": 5, "context": 4096, "window": 0, "sinks": 0, **scales, "mix": 8},
        # ragged prompt chunks behind cached context, sliding window and sinks
        {"name": "attention prompts window", "op": "attention", **heads15, "type": "bfloat16", "page": 16, "batch": 4,
         "tokens": 3500, "context": 6000, "window": 1000, "sinks": 5, **scales, "mix": 9},
        # one long prompt, fully causal: tensor-core bound
        {"name": "attention prompt 8192", "op": "attention", **heads15, "type": "float16", "page": 64, "batch": 1,
         "tokens": 8192, "context": 8192, "window": 0, "sinks": 0, **scales, "mix": 10},
        # a few samples drawn from one prompt
        {"name": "prefix 8x525", "op": "prefix", **heads15, "type": "float16", "page": 16, "batch": 8, "prefix": 525,
         "tokens": 1, "context": 64, **scales, "mix": 11},
        # a batch behind one system prompt, each with a ragged continuation of its own
        {"name": "prefix 64x8192", "op": "prefix", **heads7, "type": "bfloat16", "page": 64, "batch": 64,
         "prefix": 8192, "tokens": 1, "context": 700, **scales, "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention", "attention", "prefix"])
    heads, kv = rng.choice([(12, 2), (28, 4), (14, 2), (7, 1), (8, 8), (16, 1), (4, 1)])
    case = {"op": op, "heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128]),
            "type": rng.choice(["float16", "bfloat16"]), "page": rng.choice([16, 32, 64, 128]),
            "k_exp": rng.randrange(-4, 3), "v_exp": rng.randrange(-6, 1), "mix": rng.randrange(1 << 20)}
    if op == "append":
        tokens = rng.choice([1, 1, _spread(rng, 2, 2048)])
        batch = _spread(rng, 1, 64 if tokens == 1 else 8)
        return {**case, "batch": batch, "tokens": tokens, "context": tokens + _spread(rng, 1, 2048)}
    if op == "read":
        tokens = _spread(rng, 1, 8192)
        return {**case, "batch": _spread(rng, 1, 8), "tokens": tokens, "context": tokens + rng.choice([0, 0, rng.randrange(0, 500)])}
    if op == "prefix":
        return {**case, "batch": _spread(rng, 1, 128), "prefix": _spread(rng, 100, 16384),
                "tokens": rng.choice([1, 1, 1, 2, 3]), "context": 3 + _spread(rng, 1, 500)}
    window, sinks = rng.choice([(0, 0), (_spread(rng, 1, 2000), rng.randrange(0, 9))])
    kind = rng.choice(["decode", "decode", "drafts", "prompts"])
    if kind == "prompts":
        batch, tokens = rng.choice([1, 2, 3, 4]), _spread(rng, 2, 2500)
        context = tokens + rng.randrange(0, 2000)
    else:
        tokens = 1 if kind == "decode" else rng.randrange(2, 7)
        batch, context = _spread(rng, 1, 64), tokens + _spread(rng, 1, 8000)
    return {**case, "batch": batch, "tokens": tokens, "context": context, "window": window, "sinks": sinks}


def _sizes(case):
    """Per sequence: (new tokens, cached positions with them). The first sequence has the case's full sizes, the others
    ragged ones below it."""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["batch"]):
        new = case["tokens"] if i == 0 or case["tokens"] == 1 else rng.randint(max(1, case["tokens"] // 3), case["tokens"])
        got.append((new, case["context"] if i == 0 else max(new, rng.randint(case["context"] // 3, case["context"]))))
    return got


# ------------------------------------------------------------------------------------------------ the format, plainly
# E2M1 numbers and the borders between them; ties go to the even code, so every second border belongs to the upper one.
_NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_BORDERS = [0.25, math.nextafter(0.75, 0), 1.25, math.nextafter(1.75, 0), 2.5, math.nextafter(3.5, 0), 5.0]


def _quantise(x, power):
    """x [..., dim] of a 16-bit type -> codes uint8 [..., dim / 2] and scales uint8 [..., dim / 16]. Ratios in 64 bits: many of
    them lie on a border."""
    x = x.unflatten(-1, (-1, 16))
    scale = (x.abs().amax(-1).double() / 6 / power).clamp(max=448).float().to(torch.float8_e4m3fn)
    unit = scale.double()[..., None] * power
    ratio = torch.where(unit > 0, x.abs().double() / unit, torch.zeros_like(unit))
    code = torch.bucketize(ratio, torch.tensor(_BORDERS, dtype=torch.float64, device=x.device)).to(torch.uint8)
    code = (code + 8 * torch.signbit(x).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], scale.view(torch.uint8)


def _values(code, scale, power):
    """The numbers in 32 bits that codes [..., dim / 2] and scales [..., dim / 16] stand for."""
    table = torch.tensor(_NUMBERS + [-v for v in _NUMBERS], device=code.device)
    x = table[torch.stack([code & 15, code >> 4], -1).flatten(-2).int()]
    return (x.unflatten(-1, (-1, 16)) * (scale.view(torch.float8_e4m3fn).float() * power)[..., None]).flatten(-2)


def _parts(pool):
    """Views of a pool's codes [pages, kv heads, page, dim / 2] and scales [pages, kv heads, page, dim / 16]."""
    n, kv, page, row = pool.shape
    flat, codes = pool.view(n, kv, page * row), page * row * 8 // 9
    return flat[..., :codes].view(n, kv, page, row * 8 // 9), flat[..., codes:].view(n, kv, page, row // 9)


# ------------------------------------------------------------------------------------------------ inputs
def _pool(case, total, g, power, typ):
    """A pool whose every position holds the quantised values of normal numbers, of a size that suits the pool's power."""
    page, kv, dim = case["page"], case["kv"], case["dim"]
    pool = torch.empty(total, kv, page, dim * 9 // 16, dtype=torch.uint8, device="cuda")
    codes, scales = _parts(pool)
    step = max(1, (1 << 25) // (kv * page * dim))
    for lo in range(0, total, step):  # (a part at a time: the quantiser works in 64 bits)
        some = min(step, total - lo)
        x = torch.randn(some, kv, page, dim, generator=g, device="cuda").mul_(16 * power).to(typ)
        codes[lo:lo + some], scales[lo:lo + some] = _quantise(x, power)
    return pool


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + case["mix"])
    typ, page, dim, nq, nkv = _TYPES[case["type"]], case["page"], case["dim"], case["heads"], case["kv"]
    sizes, prefix = _sizes(case), case.get("prefix", 0)
    k_power, v_power = 2.0 ** case["k_exp"], 2.0 ** case["v_exp"]
    need, extra = [-(-n // page) for _, n in sizes], -(-prefix // page)
    total = sum(need) + extra + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(sizes), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    rows = sum(n for n, _ in sizes)
    starts = None
    if case["tokens"] > 1:
        ends = torch.tensor([n for n, _ in sizes]).cumsum(0)
        starts = torch.cat([torch.zeros(1, dtype=torch.long), ends]).to(torch.int32).cuda()
    state = {"op": case["op"], "heads": nq, "kv": nkv, "type": typ, "rows": rows, "k_power": k_power, "v_power": v_power,
             "k": _pool(case, total, g, k_power, typ), "v": _pool(case, total, g, v_power, typ), "table": table,
             "lengths": torch.tensor([n for _, n in sizes], dtype=torch.int32).cuda(), "starts": starts}
    if case["op"] == "append":
        angle = (torch.arange(case["context"], device="cuda", dtype=torch.float64)[:, None]
                 / 1e6 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        qkv = torch.randn(rows, nq + 2 * nkv, dim, generator=g, device="cuda")
        qkv[:, nq:nq + nkv] *= 16 * k_power
        qkv[:, nq + nkv:] *= 16 * v_power
        state["qkv"] = qkv.to(typ).view(rows, -1)
        return state
    if case["op"] == "read":
        return state
    # queries whose scores spread as they do in earnest (a deviation of about one), whatever the size of the keys
    state["q"] = torch.randn(rows, nq, dim, generator=g, device="cuda").div_(16 * k_power).to(typ)
    if case["op"] == "prefix":
        state["prefix"], state["prefix_table"] = prefix, order[at:at + extra].contiguous()
        return state
    state["window"], state["sinks"] = case["window"], case["sinks"]
    if case["window"] > 0:  # pages that no row of the sequence can see any more have been freed
        for b, (new, n) in enumerate(sizes):
            first, last = -(-case["sinks"] // page), max(0, n - new + 1 - case["window"]) // page
            if last > first:
                table[b, first:last] = -1
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _positions(lengths, starts, rows):
    """Sequence and cache position of every row."""
    if starts is None:
        return torch.arange(rows, device=lengths.device), lengths.long() - 1
    t = torch.arange(rows, device=lengths.device)
    seq = torch.searchsorted(starts[1:].long(), t, right=True)
    return seq, lengths.long()[seq] - (starts.long()[seq + 1] - t)


def _plain_read(s):
    seq, pos = _positions(s["lengths"], s["starts"], s["rows"])
    page = s["k"].shape[2]
    at = s["table"][seq, pos // page].long()
    (kc, ks), (vc, vs) = _parts(s["k"]), _parts(s["v"])
    place = (at, slice(None), pos % page)
    return (_values(kc[place], ks[place], s["k_power"]).to(s["type"]), _values(vc[place], vs[place], s["v_power"]).to(s["type"]))


def _plain_append(s):
    rows, page, nq, nkv, typ = s["rows"], s["k"].shape[2], s["heads"], s["kv"], s["type"]
    x = s["qkv"].view(rows, nq + 2 * nkv, -1)
    dim = x.shape[-1]
    seq, pos = _positions(s["lengths"], s["starts"], rows)
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    lo, hi = x[:, :nq, :dim // 2].float(), x[:, :nq, dim // 2:].float()
    q = torch.cat([lo * c - hi * n, hi * c + lo * n], dim=-1).to(typ)
    # the keys decide codes, so they are turned in 64 bits before their one rounding
    c, n = c.double(), n.double()
    lo, hi = x[:, nq:nq + nkv, :dim // 2].double(), x[:, nq:nq + nkv, dim // 2:].double()
    k = torch.cat([lo * c - hi * n, hi * c + lo * n], dim=-1).float().to(typ)
    place = (s["table"][seq, pos // page].long(), slice(None), pos % page)
    (kc, ks), (vc, vs) = _parts(s["k"]), _parts(s["v"])
    kc[place], ks[place] = _quantise(k, s["k_power"])
    vc[place], vs[place] = _quantise(x[:, nq + nkv:], s["v_power"])
    return (q, *_plain_read(s))


def _gather(pool, table, power):
    """[sequences, kv heads, positions, dim] in 32 bits of the pages in `table`."""
    codes, scales = _parts(pool)
    at = table.clamp(min=0).long()
    return _values(codes[at], scales[at], power).transpose(1, 2).flatten(2, 3)


def _by_sequence(s):
    """q as [sequences, kv heads, group, rows, dim] in 32 bits, padded to the longest, and which rows are real."""
    q, nkv = s["q"], s["kv"]
    n, nq, dim = q.shape
    batch = s["lengths"].shape[0]
    starts = torch.arange(batch + 1, device=q.device) if s["starts"] is None else s["starts"].long()
    most = int((starts[1:] - starts[:-1]).max())
    idx = starts[:-1, None] + torch.arange(most, device=q.device)
    real = idx < starts[1:, None]
    x = q[idx.clamp(max=n - 1)].float().view(batch, most, nkv, nq // nkv, dim)
    pos = s["lengths"].long()[:, None] - (starts[1:, None] - idx)
    return x.permute(0, 2, 3, 1, 4), real, pos


def _plain_attention(s):
    q, real, pos = _by_sequence(s)
    k, v = _gather(s["k"], s["table"], s["k_power"]), _gather(s["v"], s["table"], s["v_power"])
    j = torch.arange(k.shape[2], device=k.device)
    seen = j <= pos[..., None]
    if s["window"] > 0:
        seen &= (j > pos[..., None] - s["window"]) | (j < s["sinks"])
    score = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(q.shape[-1] ** -0.5)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v[:, :, None]) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[real].to(s["q"].dtype)


def _plain_prefix(s):
    q, real, pos = _by_sequence(s)
    scale = q.shape[-1] ** -0.5
    k, v = _gather(s["k"], s["table"], s["k_power"]), _gather(s["v"], s["table"], s["v_power"])
    own_score = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * scale
    j = torch.arange(k.shape[2], device=k.device)
    own_score.masked_fill_(~(j <= pos[..., None])[:, None, None], -math.inf)
    pk = _gather(s["k"], s["prefix_table"][None], s["k_power"])[:, :, None, :s["prefix"]]
    pv = _gather(s["v"], s["prefix_table"][None], s["v_power"])[:, :, None, :s["prefix"]]
    score = torch.cat([torch.matmul(q, pk.transpose(-1, -2)) * scale, own_score], dim=-1)
    p = (score - score.amax(-1, keepdim=True)).exp()
    out = torch.matmul(p[..., :s["prefix"]], pv) + torch.matmul(p[..., s["prefix"]:], v[:, :, None])
    out = (out / p.sum(-1, keepdim=True)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[real].to(s["q"].dtype)


_module = None


def _kernels():
    global _module
    if _module is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(1, _PACKAGE)
        from kernels import paged_fp4

        _module = paged_fp4
    return _module


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention, "prefix": _plain_prefix}[op](s)
    fp4 = _kernels()
    scales = {"k_scale": s["k_power"], "v_scale": s["v_power"]}
    if op == "attention":
        return fp4.paged_attention_fp4(s["q"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"],
                                       window=s["window"], sinks=s["sinks"], **scales)
    if op == "prefix":
        return fp4.shared_prefix_attention_fp4(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["table"],
                                               s["lengths"], starts=s["starts"], **scales)
    got = ()
    if op == "append":
        got = (fp4.paged_append_fp4(s["qkv"], s["k"], s["v"], s["table"], s["lengths"], s["cos"], s["sin"], s["heads"],
                                    s["kv"], starts=s["starts"], **scales),)
    return (*got, *fp4.paged_read_fp4(s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"], tokens=s["rows"],
                                      dtype=s["type"], **scales))


# ------------------------------------------------------------------------------------------------ work and exact values
def _seen_by(case, pos):
    """How many cached positions the row at `pos` sees."""
    if case.get("window", 0) <= 0:
        return pos + 1
    lo = max(0, pos + 1 - case["window"])
    return pos + 1 - lo + min(case["sinks"], lo)


def work(case):
    nq, nkv, dim = case["heads"], case["kv"], case["dim"]
    sizes = _sizes(case)
    rows = sum(new for new, _ in sizes)
    cached_bytes = 2 * nkv * dim * 9 // 16  # k and v of one position
    tables = 4 * (sum(n for _, n in sizes) // case["page"] + 2 * len(sizes))
    if case["op"] == "read":
        return {"bytes": rows * (cached_bytes + 2 * nkv * dim * 2) + tables, "flops": rows * 2 * nkv * dim}
    if case["op"] == "append":  # rows of q, k and v in; q, the cache's bytes and the values that were read back out
        positions = len({p for new, n in sizes for p in range(n - new, n)})
        moved = (nq + 2 * nkv) * dim * 2 + nq * dim * 2 + cached_bytes + 2 * nkv * dim * 2
        return {"bytes": rows * moved + positions * dim * 4 + tables, "flops": 3 * rows * (nq + 5 * nkv) * dim}
    pairs, cached = 0, 0
    for new, n in sizes:
        pairs += sum(_seen_by(case, p) for p in range(n - new, n))
        lo = max(0, n - new + 1 - case["window"]) if case.get("window", 0) > 0 else 0
        cached += n - lo + min(case.get("sinks", 0), lo)
    pairs += rows * case.get("prefix", 0)
    cached += case.get("prefix", 0)
    return {"bytes": cached * cached_bytes + 2 * rows * nq * dim * 2 + 4 * (cached // case["page"] + len(sizes)),
            "flops": 4 * pairs * nq * dim}


def _nearest(x, power):
    """What x [..., dim] stands for in the cache, in 64 bits, by the distances to the numbers of the format."""
    x = x.unflatten(-1, (-1, 16))
    top = x.abs().amax(-1, keepdim=True) / (6 * power)
    # E4M3: steps of 2^-3 of the power of two below, at least 2^-9; ties to even
    step = torch.exp2(torch.frexp(top.clamp(min=2.0 ** -6)).exponent.double() - 4)  # (its mantissa is in [0.5, 1))
    unit = torch.round(top / step).mul(step).clamp(max=448.0) * power
    y = torch.where(unit > 0, x.abs() / unit.clamp(min=2.0 ** -100), torch.zeros_like(x)).clamp(max=6.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))  # (each number's half step is a power of two: ties to even)
    return (torch.round(y / step) * step * unit * torch.sign(x)).flatten(-2)


def _read_exactly(pool, where, page, power, rows_of):
    """[positions, kv heads, dim] in 64 bits of the pages and offsets of `where` (a page for each position)."""
    n, kv, size, row = pool.shape
    dim, raw = row * 16 // 9, pool.view(n, kv, size * row)
    offset = rows_of % page
    byte = raw[where[:, None], :, offset[:, None] * (dim // 2) + torch.arange(dim // 2, device=pool.device)]  # [positions, bytes, kv]
    grid = raw[where[:, None], :, size * dim // 2 + offset[:, None] * (dim // 16) + torch.arange(dim // 16, device=pool.device)]
    code = torch.stack([byte % 16, byte // 16], 2).flatten(1, 2).transpose(1, 2).long()
    size_of, sign = code % 8, 1 - 2 * (code // 8)
    exponent, odd = size_of // 2, size_of % 2
    number = torch.where(exponent > 0, (1 + odd / 2.0).double() * torch.exp2(exponent.double() - 1), odd / 2.0)
    e4, m4 = (grid.long() // 8 % 16).double(), (grid.long() % 8).double()
    scale = torch.where(e4 > 0, (1 + m4 / 8) * torch.exp2(e4 - 7), m4 * 2.0 ** -9).transpose(1, 2)
    return (number * sign).double() * scale.repeat_interleave(16, -1) * power


def exact(case, seed):
    s = prepare(case, seed)
    sizes, page, dim, nkv = _sizes(case), case["page"], case["dim"], case["kv"]
    group = case["heads"] // nkv
    kp, vp = s["k_power"], s["v_power"]
    if case["op"] == "append":
        rows = s["qkv"].double().view(-1, case["heads"] + 2 * nkv, dim)
        pos = torch.cat([torch.arange(n - new, n, device="cuda") for new, n in sizes])
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        x = rows[:, :case["heads"] + nkv]
        y = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * turn
        y = torch.cat([y.real, y.imag], -1)
        k = y[:, case["heads"]:].to(s["type"]).double()  # the cache quantises what a 16-bit cache would hold
        return y[:, :case["heads"]], _nearest(k, kp), _nearest(rows[:, case["heads"] + nkv:], vp)
    if case["op"] == "read":
        outs = [], []
        for b, (new, n) in enumerate(sizes):
            pos = torch.arange(n - new, n, device="cuda")
            for some in pos.split(4096):
                where = s["table"][b].long()[some // page]
                outs[0].append(_read_exactly(s["k"], where, page, kp, some))
                outs[1].append(_read_exactly(s["v"], where, page, vp, some))
        return torch.cat(outs[0]), torch.cat(outs[1])
    out, t = [], 0
    ahead = case.get("prefix", 0)
    if ahead:
        at = torch.arange(ahead, device="cuda")
        where = s["prefix_table"].long()[at // page]
        before = _read_exactly(s["k"], where, page, kp, at), _read_exactly(s["v"], where, page, vp, at)
    for b, (new, n) in enumerate(sizes):
        at = torch.arange(n, device="cuda")
        where = s["table"][b].long().clamp(min=0)[at // page]
        k, v = _read_exactly(s["k"], where, page, kp, at), _read_exactly(s["v"], where, page, vp, at)
        if ahead:
            k, v = torch.cat([before[0], k]), torch.cat([before[1], v])
        j = torch.arange(n + ahead, device="cuda")
        for lo in range(0, new, 512):
            some = range(lo, min(new, lo + 512))
            pos = torch.arange(n - new + some[0], n - new + some[-1] + 1, device="cuda") + ahead
            hide = j[None] > pos[:, None]
            if case.get("window", 0) > 0:
                hide |= (j[None] <= pos[:, None] - case["window"]) & (j[None] >= case["sinks"])
            heads = []
            for h in range(case["heads"]):
                q = s["q"][t + some[0]:t + some[-1] + 1, h].double()
                a = torch.einsum("td,jd->tj", q, k[:, h // group]) / math.sqrt(dim)
                heads.append(torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v[:, h // group])
            out.append(torch.stack(heads, 1))
        t += new
    return torch.cat(out)
