"""Several samples of one prompt on a paged cache (kernels.e2e.sample) against the runner's own forward pass, which keeps a
contiguous cache and attends with SDPA: the logits that every sample's tokens were picked from, and their log
probabilities."""

import pytest
import torch

transformers = pytest.importorskip("transformers")

ARCH = dict(vocab_size=1000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=8,
            num_key_value_heads=2, head_dim=64, tie_word_embeddings=True, rms_norm_eps=1e-6, rope_theta=1e6,
            max_position_embeddings=512)


def _runner(backend, dtype=torch.float16):
    from kernels.e2e.model import QwenRunner, make_backend, random_qwen2

    return QwenRunner(random_qwen2(ARCH, dtype=dtype), make_backend(backend), max_len=256)


def _full_logits(runner, ids, window, sinks):
    """Logits [T, V] of the runner's forward pass of one sequence (SDPA over the whole cache, masked)."""
    if window == 0:
        return runner.forward(ids[None], torch.arange(len(ids), device="cuda"), all_logits=True)[0]
    keep = torch.nn.functional.scaled_dot_product_attention

    def masked(q, k, v, attn_mask=None, **more):
        pos, j = torch.arange(q.shape[2], device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
        return keep(q, k, v, attn_mask=attn_mask & ((j > pos - window) | (j < sinks)), **more)

    torch.nn.functional.scaled_dot_product_attention = masked
    try:
        return runner.forward(ids[None], torch.arange(len(ids), device="cuda"), all_logits=True)[0]
    finally:
        torch.nn.functional.scaled_dot_product_attention = keep


@pytest.mark.gpu
@pytest.mark.parametrize("backend,prompt,window,sinks", [("fp16", 37, 0, 0), ("ours", 100, 0, 0), ("fp16", 64, 20, 3),
                                                         ("ours", 75, 30, 2)])
def test_samples_match_the_runner(backend, prompt, window, sinks):
    from kernels import _lib
    from kernels.e2e.sample import PagedSampler

    runner = _runner(backend)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 1000, (prompt,), generator=g, device="cuda")
    seen = []

    def pick(logits):
        seen.append(logits.clone())
        return torch.randint(0, 1000, (logits.shape[0],), generator=g, device="cuda")

    sampler = PagedSampler(runner, 3, 128, 40, page_size=16, window=window, sinks=sinks)
    _lib.clear_device_error()
    out = sampler.generate(ids, 24, pick, top=4)
    assert _lib.device_error() == 0
    assert out["tokens"].shape == out["logprobs"].shape == out["entropy"].shape == (3, 24)
    assert out["top_ids"].shape == (3, 24, 4)
    for b in range(3):
        want = _full_logits(runner, torch.cat([ids, out["tokens"][b, :-1]]), window, sinks)[prompt - 1:]
        got = torch.stack([x[b] for x in seen])
        # two layers of fp16 arithmetic in another order: the runner's own tolerance for its fused decode path
        torch.testing.assert_close(got.float(), want.float(), atol=5e-2, rtol=5e-2)
        logp = torch.log_softmax(got.double(), -1)
        torch.testing.assert_close(out["logprobs"][b].double(), logp.gather(1, out["tokens"][b][:, None])[:, 0], atol=1e-5, rtol=1e-6)
        assert torch.equal(out["top_ids"][b], torch.sort(got.float(), dim=-1, descending=True, stable=True)[1][:, :4])


@pytest.mark.gpu
def test_refusals():
    from kernels.e2e.sample import PagedSampler

    sampler = PagedSampler(_runner("fp16"), 2, 16, 8, page_size=16)
    with pytest.raises(ValueError):
        sampler.prefill(torch.zeros(17, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        sampler.generate(torch.zeros(4, dtype=torch.long, device="cuda"), 9)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 6])
def test_steps_are_counted(window):
    """A step without a prompt, or past max_new, is refused before it changes anything; a new prompt starts the count again."""
    from kernels.e2e.sample import PagedSampler

    sampler = PagedSampler(_runner("fp16"), 2, 16, 3, page_size=16, window=window, sinks=1)
    token = torch.zeros(2, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError):
        sampler.step(token)
    for prompt in (4, 16):
        sampler.prefill(torch.arange(prompt, device="cuda"))
        for _ in range(3):
            assert sampler.step(token).isfinite().all()
        lengths = sampler.lengths.clone()
        with pytest.raises(ValueError):
            sampler.step(token)
        assert torch.equal(sampler.lengths, lengths)


@pytest.mark.gpu
@pytest.mark.parametrize("prompt,window,sinks,dtype", [(75, 0, 0, torch.float16), (64, 20, 3, torch.bfloat16)])
def test_samples_on_a_4_bit_cache(prompt, window, sinks, dtype):
    """The same sampler on 4-bit pages. In every layer and step its attention gives, to the rounding of the output and of the
    probabilities, what 64-bit attention gives on the values that its pages hold; a captured step gives the eager one's logits."""
    from _paged_fp4 import NUMBERS, SCALES, unpack
    from kernels import _lib
    from kernels.e2e.sample import PagedSampler

    runner = _runner("fp16", dtype)
    ids = torch.arange(prompt, device="cuda") * 7 % 1000
    scales = {"k_scale": 0.25, "v_scale": 2.0 ** -5}
    sampler = PagedSampler(runner, 3, 128, 40, page_size=16, window=window, sinks=sinks, cache="fp4", **scales)

    def values(pool, power):
        codes, grid = unpack(pool.cpu())
        unit = SCALES[grid.clamp(max=126)].repeat_interleave(16, -1) * power  # (no NaN is ever appended here)
        return NUMBERS[codes % 8] * torch.where(codes > 7, -1.0, 1.0) * unit

    checked = []
    attend, behind = sampler.attention, sampler.behind_prefix

    def check(q, k, v, tables, positions, out):
        k, v = values(k, scales["k_scale"]), values(v, scales["v_scale"])
        for t, (table, n) in enumerate(zip(tables, positions)):
            j = torch.arange(n)
            ks, vs = (x[table.cpu().long()[j // 16], :, j % 16].repeat_interleave(4, 1) for x in (k, v))
            see = torch.ones(n, dtype=torch.bool) if window == 0 else (j >= n - window) | (j < sinks)
            score = torch.einsum("hd,jhd->hj", q[t].double().cpu(), ks[see]) * 64 ** -0.5
            p = torch.softmax(score, -1)
            want, spread = torch.einsum("hj,jhd->hd", p, vs[see]), torch.einsum("hj,jhd->hd", p, vs[see].abs())
            u = torch.finfo(dtype).eps / 2
            tol = u * want.abs() + (u + 2.0 ** -13) * spread + n * 2.0 ** -25 * vs.abs().max()
            assert ((out[t].double().cpu() - want).abs() <= tol).all()
        checked.append(len(out))

    def attention(q, k, v, table, lengths, starts=None, **more):
        out = attend(q, k, v, table, lengths, starts=starts, **more)
        if starts is None:
            check(q, k, v, table, lengths.tolist(), out)
        else:
            rows = range(0, prompt, 13)
            check(q[rows], k, v, table.expand(len(rows), -1), [r + 1 for r in rows], out[rows])
        return out

    def behind_prefix(q, k, v, prefix_table, n, table, lengths):
        out = behind(q, k, v, prefix_table, n, table, lengths)
        kv = values(k, scales["k_scale"]), values(v, scales["v_scale"])
        for b, own in enumerate(lengths.tolist()):
            i, j = torch.arange(n), torch.arange(own)
            ks, vs = (torch.cat([x[prefix_table.cpu().long()[i // 16], :, i % 16], x[table[b].cpu().long()[j // 16], :, j % 16]])
                      .repeat_interleave(4, 1) for x in kv)
            p = torch.softmax(torch.einsum("hd,jhd->hj", q[b].double().cpu(), ks) * 64 ** -0.5, -1)
            want, spread = torch.einsum("hj,jhd->hd", p, vs), torch.einsum("hj,jhd->hd", p, vs.abs())
            u = torch.finfo(dtype).eps / 2
            assert ((out[b].double().cpu() - want).abs() <= u * want.abs() + (u + 2.0 ** -13) * spread
                    + (n + own) * 2.0 ** -25 * vs.abs().max()).all()
        checked.append(len(out))
        return out

    sampler.attention, sampler.behind_prefix = attention, behind_prefix
    _lib.clear_device_error()
    g = torch.Generator(device="cuda").manual_seed(1)
    out = sampler.generate(ids, 12, lambda logits: torch.randint(0, 1000, (logits.shape[0],), generator=g, device="cuda"), top=2)
    assert _lib.device_error() == 0 and len(checked) == 2 * 12
    assert out["tokens"].shape == (3, 12) and out["logprobs"].isfinite().all()
    sampler.attention, sampler.behind_prefix = attend, behind
    token = out["tokens"][:, -1].contiguous()
    state = sampler.k.clone(), sampler.v.clone(), sampler.lengths.clone()
    sampler.step(token)  # (allocates what a step needs before the capture)
    for x, y in zip((sampler.k, sampler.v, sampler.lengths), state):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = sampler.step(token)
    for x, y in zip((sampler.k, sampler.v, sampler.lengths), state):
        x.copy_(y)
    graph.replay()
    kept = captured.clone()
    for x, y in zip((sampler.k, sampler.v, sampler.lengths), state):
        x.copy_(y)
    assert torch.equal(sampler.step(token), kept)


def test_a_cache_of_another_kind_is_refused():
    from kernels.e2e.sample import PagedSampler

    class Runner:
        tp = None

    with pytest.raises(ValueError, match="16 or fp4"):
        PagedSampler(Runner(), 2, 16, 8, cache="8")
