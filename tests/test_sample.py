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
