"""Workloads of the paged-cache serving operators, for timing and for comparing outputs.

Four operators that a batch server runs around the projections of a decoder:

* `append`    rotate q and k by their positions and write k and v into a paged cache;
* `attention` attention over the pages, causal, optionally limited to a sliding window plus a few first
              tokens that stay visible; one token per sequence (decode) or ragged rows of them (prompts);
* `prefix`    attention of a batch whose sequences share a long prefix, computed once for all of them;
* `logprobs`  log probabilities of given tokens, with the entropy and the top alternatives.

`run` computes them in plain torch, in 32 bits and rounded once at the end, or with `own = True` by the
`kernels` package. Head layouts are those of kernels/config.py (12 query / 2 kv heads and 28 / 4, head_dim 128)
and their tensor-parallel shards; vocabularies and prompt lengths likewise.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "llm-decode-kernels_b200")
_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    heads15 = {"heads": 12, "kv": 2, "dim": 128}
    heads7 = {"heads": 28, "kv": 4, "dim": 128}
    return [
        # one decode step of a batch server: one new token for each of 64 sequences
        {"name": "append decode 64", "op": "append", **heads7, "type": "float16", "page": 64, "batch": 64,
         "tokens": 1, "context": 2048, "mix": 1},
        # the prompts of a batch, ragged, appended in one call (the second half of each prompt: chunked prefill)
        {"name": "append prompts", "op": "append", **heads7, "type": "bfloat16", "page": 16, "batch": 8,
         "tokens": 2048, "context": 4096, "mix": 2},
        # interactive decode of one sequence at the benchmark's prompt length: latency
        {"name": "attention decode 1x640", "op": "attention", **heads15, "type": "float16", "page": 16, "batch": 1,
         "tokens": 1, "context": 640, "window": 0, "sinks": 0, "mix": 3},
        # decode of a full batch over ragged contexts: bandwidth
        {"name": "attention decode 64x8192", "op": "attention", **heads7, "type": "bfloat16", "page": 64, "batch": 64,
         "tokens": 1, "context": 8192, "window": 0, "sinks": 0, "mix": 4},
        # long conversations decoded through a window with sink tokens; pages outside it are already freed
        {"name": "attention decode window", "op": "attention", **heads15, "type": "float16", "page": 32, "batch": 48,
         "tokens": 1, "context": 32768, "window": 1024, "sinks": 4, "mix": 5},
        # ragged prompt chunks behind cached context, sliding window and sinks
        {"name": "attention prompts window", "op": "attention", **heads15, "type": "bfloat16", "page": 16, "batch": 4,
         "tokens": 3500, "context": 6000, "window": 1000, "sinks": 5, "mix": 6},
        # one long prompt, fully causal: tensor-core bound
        {"name": "attention prompt 8192", "op": "attention", **heads15, "type": "float16", "page": 64, "batch": 1,
         "tokens": 8192, "context": 8192, "window": 0, "sinks": 0, "mix": 7},
        # a few samples drawn from one prompt
        {"name": "prefix 8x525", "op": "prefix", **heads15, "type": "float16", "page": 16, "batch": 8, "prefix": 525,
         "tokens": 1, "context": 64, "mix": 8},
        # a batch behind one system prompt, each with a ragged continuation of its own
        {"name": "prefix 64x8192", "op": "prefix", **heads7, "type": "bfloat16", "page": 64, "batch": 64,
         "prefix": 8192, "tokens": 1, "context": 700, "mix": 9},
        # a large batch of questions about one long document
        {"name": "prefix 200x32001", "op": "prefix", **heads15, "type": "float16", "page": 128, "batch": 200,
         "prefix": 32001, "tokens": 1, "context": 300, "mix": 10},
        # the pick of one decode step, with five alternatives: latency
        {"name": "logprobs 1", "op": "logprobs", "type": "float16", "rows": 1, "vocab": 151936, "top": 5, "mix": 11},
        # scoring a prompt's tokens, with twenty alternatives each: bandwidth
        {"name": "logprobs 2048", "op": "logprobs", "type": "bfloat16", "rows": 2048, "vocab": 152064, "top": 20,
         "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "prefix", "logprobs"])
    kind = rng.choice(["float16", "bfloat16"])
    mix = rng.randrange(1 << 20)
    if op == "logprobs":
        rows = _spread(rng, 1, 1500)
        return {"op": op, "type": rng.choice(["float16", "bfloat16", "float32"]), "rows": rows,
                "vocab": _spread(rng, 1000, 152064), "top": rng.choice([0, 1, 5, 20, 32]), "mix": mix}
    heads, kv = rng.choice([(12, 2), (28, 4), (14, 2), (7, 1), (8, 8), (16, 1), (4, 1)])
    case = {"op": op, "heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128]), "type": kind,
            "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        tokens = rng.choice([1, 1, _spread(rng, 2, 2048)])
        batch = _spread(rng, 1, 64 if tokens == 1 else 8)
        return {**case, "batch": batch, "tokens": tokens, "context": tokens + _spread(rng, 1, 2048), "mix": mix}
    if op == "prefix":
        return {**case, "batch": _spread(rng, 1, 128), "prefix": _spread(rng, 100, 16384),
                "tokens": rng.choice([1, 1, 1, 2, 3]), "context": 3 + _spread(rng, 1, 500), "mix": mix}
    window, sinks = rng.choice([(0, 0), (_spread(rng, 1, 2000), rng.randrange(0, 9))])
    if rng.random() < 0.6:  # one token each
        batch = _spread(rng, 1, 64)
        return {**case, "batch": batch, "tokens": 1, "context": _spread(rng, 1, 8192), "window": window,
                "sinks": sinks, "mix": mix}
    batch = rng.choice([1, 2, 3, 4])
    tokens = _spread(rng, 2, 2500)
    return {**case, "batch": batch, "tokens": tokens, "context": tokens + rng.randrange(0, 2000), "window": window,
            "sinks": sinks, "mix": mix}


def _sizes(case):
    """Per sequence: (new tokens, cached positions with them). The first sequence has the case's full sizes, the others
    ragged ones below it."""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["batch"]):
        new = case["tokens"] if i == 0 or case["tokens"] == 1 else rng.randint(max(1, case["tokens"] // 3), case["tokens"])
        got.append((new, case["context"] if i == 0 else max(new, rng.randint(case["context"] // 3, case["context"]))))
    return got


# ------------------------------------------------------------------------------------------------ inputs
def _pages(case, lengths, extra, g, typ):
    """Page tables of `lengths` (out of a shuffled pool) and the pools of k and v; `extra` pages more for a prefix."""
    page, kv, dim = case["page"], case["kv"], case["dim"]
    need = [-(-n // page) for n in lengths]
    wide = max(need) + 1
    total = sum(need) + extra + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    k = torch.randn(total, kv, page, dim, generator=g, device="cuda", dtype=typ)
    v = torch.randn(total, kv, page, dim, generator=g, device="cuda", dtype=typ)
    return table, order[at:at + extra].contiguous(), k, v


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + case["mix"])
    typ = _TYPES[case["type"]]
    if case["op"] == "logprobs":
        logits = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda", dtype=typ).mul_(3)
        targets = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda")
        return {"op": "logprobs", "logits": logits, "targets": targets, "top": case["top"]}
    sizes = _sizes(case)
    prefix = case.get("prefix", 0)
    lengths = [n for _, n in sizes]
    page, dim = case["page"], case["dim"]
    table, prefix_table, k, v = _pages(case, lengths, -(-prefix // page), g, typ)
    rows = sum(n for n, _ in sizes)
    starts = None
    if case["tokens"] > 1:
        ends = torch.tensor([n for n, _ in sizes]).cumsum(0)
        starts = torch.cat([torch.zeros(1, dtype=torch.long), ends]).to(torch.int32).cuda()
    state = {"op": case["op"], "heads": case["heads"], "kv": case["kv"], "k": k, "v": v, "table": table,
             "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(), "starts": starts}
    if case["op"] == "append":
        angle = (torch.arange(case["context"], device="cuda", dtype=torch.float64)[:, None]
                 / 1e6 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim))
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        state["qkv"] = torch.randn(rows, (case["heads"] + 2 * case["kv"]) * dim, generator=g, device="cuda", dtype=typ)
        return state
    state["q"] = torch.randn(rows, case["heads"], dim, generator=g, device="cuda", dtype=typ)
    if case["op"] == "prefix":
        state["prefix"], state["prefix_table"] = prefix, prefix_table
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


def _plain_append(s):
    rows, page, dim = s["qkv"].shape[0], s["k"].shape[2], s["k"].shape[3]
    nq, nkv = s["heads"], s["kv"]
    seq, pos = _positions(s["lengths"], s["starts"], rows)
    x = s["qkv"].view(rows, nq + 2 * nkv, dim)
    lo, hi = x[:, :nq + nkv, :dim // 2].float(), x[:, :nq + nkv, dim // 2:].float()
    c, n = s["cos"][pos][:, None].float(), s["sin"][pos][:, None].float()
    turned = torch.cat([lo * c - hi * n, hi * c + lo * n], dim=-1).to(x.dtype)
    at = s["table"][seq, pos // page].long()
    s["k"][at, :, pos % page] = turned[:, nq:]
    s["v"][at, :, pos % page] = x[:, nq + nkv:]
    return turned[:, :nq].contiguous(), s["k"], s["v"]


def _gather(pool, table):
    """[sequences, kv heads, positions, dim] in 32 bits of the pages in `table`."""
    x = pool[table.clamp(min=0).long()].float()
    return x.transpose(1, 2).flatten(2, 3)


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
    k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
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
    k, v = _gather(s["k"], s["table"]), _gather(s["v"], s["table"])
    own_score = torch.matmul(q, k[:, :, None].transpose(-1, -2)) * scale
    j = torch.arange(k.shape[2], device=k.device)
    own_score.masked_fill_(~(j <= pos[..., None])[:, None, None], -math.inf)
    pk, pv = (_gather(s[n], s["prefix_table"][None])[:, :, None, :s["prefix"]] for n in ("k", "v"))
    score = torch.cat([torch.matmul(q, pk.transpose(-1, -2)) * scale, own_score], dim=-1)
    p = (score - score.amax(-1, keepdim=True)).exp()
    out = torch.matmul(p[..., :s["prefix"]], pv) + torch.matmul(p[..., s["prefix"]:], v[:, :, None])
    out = (out / p.sum(-1, keepdim=True)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[real].to(s["q"].dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    entropy = (lse - (e * x).sum(-1, keepdim=True) / total)[:, 0]
    logprob = (x.gather(1, s["targets"][:, None]) - lse)[:, 0]
    value, index = torch.sort(x, dim=-1, descending=True, stable=True)
    return logprob, entropy, value[:, :s["top"]] - lse, index[:, :s["top"]].contiguous()


_modules = None


def _kernels():
    global _modules
    if _modules is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(1, _PACKAGE)
        from kernels import logprobs, paged

        _modules = paged, logprobs
    return _modules


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "prefix": _plain_prefix,
                "logprobs": _plain_logprobs}[op](s)
    paged, logprobs = _kernels()
    if op == "append":
        q = paged.paged_append(s["qkv"], s["k"], s["v"], s["table"], s["lengths"], s["cos"], s["sin"], s["heads"],
                               s["kv"], starts=s["starts"])
        return q, s["k"], s["v"]
    if op == "attention":
        return paged.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], starts=s["starts"],
                                     window=s["window"], sinks=s["sinks"])
    if op == "prefix":
        return paged.shared_prefix_attention(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["table"],
                                             s["lengths"], starts=s["starts"])
    return logprobs.token_logprobs(s["logits"], s["targets"], top=s["top"])


# ------------------------------------------------------------------------------------------------ work and exact values
def _seen_by(case, pos):
    """How many cached positions the row at `pos` sees."""
    if case.get("window", 0) <= 0:
        return pos + 1
    lo = max(0, pos + 1 - case["window"])
    return pos + 1 - lo + min(case["sinks"], lo)


def work(case):
    if case["op"] == "logprobs":
        rows, vocab, size = case["rows"], case["vocab"], 4 if case["type"] == "float32" else 2
        return {"bytes": rows * (vocab * size + 8 + 8 + 12 * case["top"]), "flops": 6 * rows * vocab}
    nq, nkv, dim = case["heads"], case["kv"], case["dim"]
    sizes = _sizes(case)
    rows = sum(new for new, _ in sizes)
    if case["op"] == "append":
        positions = len({p for new, n in sizes for p in range(n - new, n)})
        return {"bytes": 2 * rows * (nq + 2 * nkv) * dim * 2 + positions * dim * 4 + 8 * len(sizes),
                "flops": 3 * rows * (nq + nkv) * dim}
    pairs, cached = 0, 0
    for new, n in sizes:
        pairs += sum(_seen_by(case, p) for p in range(n - new, n))
        lo = max(0, n - new + 1 - case["window"]) if case.get("window", 0) > 0 else 0
        cached += n - lo + min(case.get("sinks", 0), lo)
    pairs += rows * case.get("prefix", 0)
    cached += case.get("prefix", 0)
    return {"bytes": cached * nkv * dim * 2 * 2 + 2 * rows * nq * dim * 2 + 4 * (cached // case["page"] + len(sizes)),
            "flops": 4 * pairs * nq * dim}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        outs = [], [], [], []
        for x, t in zip(s["logits"].double().split(64), s["targets"].split(64)):
            logp = torch.log_softmax(x, -1)
            outs[0].append(logp[torch.arange(len(t), device=t.device), t])
            outs[1].append(-(logp.exp() * logp).sum(-1))
            outs[2].append(torch.sort(logp, dim=-1, descending=True)[0][:, :s["top"]])
        return torch.cat(outs[0]), torch.cat(outs[1]), torch.cat(outs[2]), None
    sizes, page, dim, nkv = _sizes(case), case["page"], case["dim"], case["kv"]
    group = case["heads"] // nkv
    if case["op"] == "append":
        rows = s["qkv"].double().view(-1, case["heads"] + 2 * nkv, dim)
        k, v = s["k"].double(), s["v"].double()
        q, t = [], 0
        for b, (new, n) in enumerate(sizes):
            pos = torch.arange(n - new, n, device="cuda")
            turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
            x = rows[t:t + new, :case["heads"] + nkv]
            y = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * turn
            y = torch.cat([y.real, y.imag], -1)
            q.append(y[:, :case["heads"]])
            where = s["table"][b].long()[pos // page]
            k[where, :, pos % page] = y[:, case["heads"]:]
            v[where, :, pos % page] = rows[t:t + new, case["heads"] + nkv:]
            t += new
        return torch.cat(q), k, v
    out, t = [], 0
    before = s["prefix_table"].long() if case["op"] == "prefix" else None
    ahead = case.get("prefix", 0)
    for b, (new, n) in enumerate(sizes):
        where = torch.arange(n, device="cuda")
        pages = s["table"][b].long().clamp(min=0)[where // page]
        k, v = s["k"][pages, :, where % page], s["v"][pages, :, where % page]
        if before is not None:
            at = torch.arange(ahead, device="cuda")
            k = torch.cat([s["k"][before[at // page], :, at % page], k])
            v = torch.cat([s["v"][before[at // page], :, at % page], v])
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
                a = torch.einsum("td,jd->tj", q, k[:, h // group].double()) / math.sqrt(dim)
                heads.append(torch.softmax(a.masked_fill(hide, -math.inf), -1) @ v[:, h // group].double())
            out.append(torch.stack(heads, 1))
        t += new
    return torch.cat(out)
