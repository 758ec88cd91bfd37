"""Several continuations of one prompt with the log probabilities of their tokens, on a paged cache.

The prompt runs once, in one call per layer of `paged_append` and `paged_attention`, into pages that all samples share.
Each step then appends every sample's token to pages of its own and attends with `shared_prefix_attention`, which reads
the prompt's keys and values once for all samples, or with a window with `paged_attention` (window, sinks) over page
tables that list the shared pages first. With a cache held in 4 bits the same runs on the ops of `kernels.paged_fp4`, from
the same projections. `token_logprobs` scores the picked tokens. The projections are the runner's
backend (kernels.e2e.model). The reference decodes one sequence, or a batch with a cache each
(kernels/e2e/model.py:192, 216-253); it has no counterpart of this.

    python -m kernels.e2e.sample --layers 4 --samples 16 --prompt 2048 --steps 32 [--cache fp4]
"""

from __future__ import annotations

import argparse
import functools
import time

import torch
import torch.nn.functional as F

from kernels.logprobs import token_logprobs
from kernels.paged import paged_append, paged_attention, shared_prefix_attention
from kernels.paged_fp4 import fp4_pages, paged_append_fp4, paged_attention_fp4, shared_prefix_attention_fp4


class PagedSampler:
    """`samples` continuations of a prompt of up to max_prompt tokens, each of up to max_new tokens, by a QwenRunner's
    weights (fp16 or bf16, head_dim 64 or 128, one GPU). window > 0 limits attention to the last `window` positions and
    the first `sinks`. cache: "16" in the weights' type, "fp4" in 4 bits, with the powers of two k_scale and v_scale of
    kernels.paged_fp4."""

    def __init__(self, runner, samples: int, max_prompt: int, max_new: int, page_size: int = 64, window: int = 0,
                 sinks: int = 0, cache: str = "16", k_scale: float = 1.0, v_scale: float = 1.0):
        if runner.tp is not None:
            raise ValueError("PagedSampler: one GPU (the runner is tensor parallel)")
        if cache not in ("16", "fp4"):
            raise ValueError(f"PagedSampler: a cache of {cache} (16 or fp4)")
        self.r, self.n, self.page, self.window, self.sinks = runner, samples, page_size, window, sinks
        self.max_prompt, self.max_new = max_prompt, max_new
        dev = runner.embed.device
        shared = -(-max_prompt // page_size)
        own = -(-max_new // page_size) + 1  # one more: with a window the prompt's last, partly filled page is copied
        pages = shared + samples * own
        if cache == "fp4":
            self.k = fp4_pages(len(runner.layers) * pages, runner.n_kv, page_size, runner.head_dim, dev).unflatten(0, (-1, pages))
            scales = {"k_scale": k_scale, "v_scale": v_scale}
            ops = paged_append_fp4, paged_attention_fp4, shared_prefix_attention_fp4
            self.append, self.attention, self.behind_prefix = (functools.partial(op, **scales) for op in ops)
        else:
            shape = (len(runner.layers), pages, runner.n_kv, page_size, runner.head_dim)
            self.k = torch.empty(shape, dtype=runner.embed.dtype, device=dev)
            self.append, self.attention, self.behind_prefix = paged_append, paged_attention, shared_prefix_attention
        self.v = torch.empty_like(self.k)
        self.prompt_table = torch.arange(shared, dtype=torch.int32, device=dev)
        self.own_table = torch.arange(shared, pages, dtype=torch.int32, device=dev).view(samples, own)
        positions = torch.arange(max_prompt + max_new, device=dev)
        angle = positions[:, None].float() * runner.inv_freq[None, :]
        self.cos, self.sin = angle.cos(), angle.sin()
        self.prompt = 0
        self.left = 0  # tokens that each sample may still be fed; none before a prompt
        self.lengths = torch.zeros(samples, dtype=torch.int32, device=dev)

    def _layers(self, x, attend):
        """The decoder layers over token rows x [T, hidden]; attend(layer, qkv) -> [T, n_heads * head_dim]."""
        r, be = self.r, self.r.backend
        h, residual = x, None
        for i, L in enumerate(r.layers):
            qkv, new = be.norm_linear(h, L.ln1, r.eps, residual, L.qkv)
            residual = x if residual is None else new
            act, residual = be.norm_gate_up_act(be.linear(attend(i, qkv), L.o), L.ln2, r.eps, residual, L.gate_up)
            h = be.linear(act, L.down)
        h, _ = be.norm(h, r.final_norm, r.eps, residual=residual)
        return h

    def _logits(self, h):
        r = self.r
        return F.linear(h, r.lm_head) if r.head_q is None else r.backend.linear(h, r.head_q)

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor) -> torch.Tensor:
        """Run the prompt ids [P] into the shared pages; the logits [V] after its last token."""
        r, P = self.r, ids.shape[0]
        if not 1 <= P <= self.max_prompt:
            raise ValueError(f"PagedSampler: a prompt of {P} tokens (1..{self.max_prompt})")
        starts = torch.tensor([0, P], dtype=torch.int32, device=ids.device)
        length, table = starts[1:], self.prompt_table[None]

        def attend(i, qkv):
            q = self.append(qkv, self.k[i], self.v[i], table, length, self.cos, self.sin, r.n_heads, r.n_kv, starts=starts)
            return self.attention(q, self.k[i], self.v[i], table, length, starts=starts, window=self.window,
                                  sinks=self.sinks).view(P, -1)

        h = self._layers(F.embedding(ids, r.embed), attend)
        self.prompt, self.left = P, self.max_new
        if self.window > 0:  # positions go on where the prompt ends: its full pages are shared, the rest of it is copied
            full = P // self.page
            self.table = torch.cat([self.prompt_table[:full].expand(self.n, full), self.own_table], 1)
            if P % self.page:
                for pool in (self.k, self.v):
                    pool[:, self.own_table[:, 0].long()] = pool[:, full:full + 1]
            self.lengths.fill_(P)
        else:
            self.table = self.own_table
            self.lengths.zero_()
        return self._logits(h[-1:])[0]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Feed one token to each sample (tokens int64 [n]), up to max_new times after a prompt; the logits [n, V] after it."""
        r = self.r
        if self.left <= 0:
            raise ValueError(f"PagedSampler: prefill a prompt first, and feed at most {self.max_new} tokens after it")
        self.left -= 1
        self.lengths += 1
        offset = 0 if self.window > 0 else self.prompt

        def attend(i, qkv):
            k, v = self.k[i], self.v[i]
            q = self.append(qkv, k, v, self.table, self.lengths, self.cos, self.sin, r.n_heads, r.n_kv, offset=offset)
            if self.window > 0:
                out = self.attention(q, k, v, self.table, self.lengths, window=self.window, sinks=self.sinks)
            else:
                out = self.behind_prefix(q, k, v, self.prompt_table, self.prompt, self.table, self.lengths)
            return out.view(self.n, -1)

        return self._logits(self._layers(F.embedding(tokens, r.embed), attend))

    def generate(self, ids: torch.Tensor, steps: int, pick=None, top: int = 0) -> dict:
        """`steps` tokens for each sample after the prompt ids [P]. pick(logits [n, V]) -> tokens int64 [n]; None: greedy.
        Returns tokens, logprobs, entropy [n, steps], and top_logprobs, top_ids [n, steps, top]."""
        if steps > self.max_new:
            raise ValueError(f"PagedSampler: {steps} steps (at most {self.max_new})")
        pick = pick or (lambda logits: logits.argmax(-1))
        logits = self.prefill(ids).expand(self.n, -1).contiguous()
        got = []
        for i in range(steps):
            tokens = pick(logits)
            got.append((tokens, *token_logprobs(logits, tokens, top)))
            if i + 1 < steps:
                logits = self.step(tokens)
        names = ("tokens", "logprobs", "entropy", "top_logprobs", "top_ids")
        return {name: torch.stack(column, 1) for name, column in zip(names, zip(*got))}


def main():
    from kernels import config
    from kernels.e2e.model import QwenRunner, make_backend, random_qwen2

    ap = argparse.ArgumentParser(description="Sample continuations of a random prompt on the Qwen2.5-1.5B architecture "
                                             "(random weights) and print their log probabilities.")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--backend", default="ours")
    ap.add_argument("--cache", default="16", choices=("16", "fp4"))
    a = ap.parse_args()
    model = random_qwen2({**config.QWEN15, "num_hidden_layers": a.layers})
    runner = QwenRunner(model, make_backend(a.backend), max_len=64)
    sampler = PagedSampler(runner, a.samples, a.prompt, a.steps, window=a.window, sinks=a.sinks, cache=a.cache)
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, config.QWEN15["vocab_size"], (a.prompt,), generator=g, device="cuda")

    def pick(logits):
        u = torch.rand(logits.shape, generator=g, device=logits.device)
        return (logits.float() - (-u.log()).log()).argmax(-1)

    sampler.generate(ids, min(2, a.steps), pick)  # warm-up
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = sampler.generate(ids, a.steps, pick, top=3)
    torch.cuda.synchronize()
    print(f"{a.samples} samples x {a.steps} tokens after {a.prompt}: {1e3 * (time.perf_counter() - t):.1f} ms")
    for b in range(min(4, a.samples)):
        row = ", ".join(f"{tok}:{lp:.2f}" for tok, lp in zip(out["tokens"][b, :8].tolist(), out["logprobs"][b, :8].tolist()))
        print(f"  sample {b}: {row} ...")


if __name__ == "__main__":
    main()
