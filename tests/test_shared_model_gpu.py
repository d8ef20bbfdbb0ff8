"""The model on the shared-row operators: samples forked from one prompt, recorded log
probabilities, scoring, and non-causal attention over pages.

bf16 tolerance of whole-model logits: as the other model tests compare backends (0.1 on logits of
order 1 at these widths, two layers of bf16 roundings)."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M(iva):
    from importlib import import_module
    return import_module("iva_amd.model")


def model_of(M, dev, dtype=torch.bfloat16, **kw):
    base = dict(d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, seq_len=512, dropout=0.0,
                attn_impl="hip_paged")
    base.update(kw)
    torch.manual_seed(0)
    return M.Transformer(M.TransformerConfig(**base)).to(dev, dtype).eval()


@pytest.mark.parametrize("kw", [{}, {"kv_cache_dtype": "fp8"}, {"rope_in_attention": True},
                                {"sliding_window": 1000, "sink_tokens": 4}, {"sliding_window": 40}],
                         ids=["bf16", "fp8", "rope", "wide-window", "window"])
def test_forked_decode_equals_separate_sequences(M, dev, monkeypatch, kw):
    """Two prompts, three samples each, ten different tokens: through the shared pages, and as
    six separate sequences without sharing."""
    monkeypatch.setattr(M, "SHARED_MIN_BYTES", 0)
    monkeypatch.setattr(M, "SHARED_MIN_TOKENS", 0)
    model = model_of(M, dev, **kw)
    gen = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, 512, (2, 83), generator=gen).to(dev)
    more = torch.randint(0, 512, (6, 10), generator=gen).to(dev)
    with torch.no_grad():
        cache = model.new_kv_cache(2, 93, samples=3, prompt_len=83)
        model(prompt, kv_cache=cache)
        cache.fork(3)
        alone = model.new_kv_cache(6, 93)
        model(prompt.repeat_interleave(3, dim=0), kv_cache=alone)
        assert alone.shared is None and cache.shared is not None
        for t in range(10):
            a = model(more[:, t:t + 1], kv_cache=cache)["logits"].float()
            b = model(more[:, t:t + 1], kv_cache=alone)["logits"].float()
            assert (a - b).abs().max() <= 0.1, t
        assert cache.resident_pages() >= alone.resident_pages() > 0  # (counted per sequence)
        if not kw.get("sliding_window"):
            assert cache.pool.num_pages < alone.pool.num_pages


@pytest.mark.parametrize("use_graph", [False, True], ids=["eager", "graph"])
def test_generate_samples_and_logprobs(M, dev, monkeypatch, use_graph):
    """Greedy samples equal the single continuation, log probabilities and tops are those of a
    scoring pass over the generated sequence; shared pages taken and not."""
    model = model_of(M, dev, dtype=torch.float16)
    ids = torch.randint(0, 512, (2, 50), generator=torch.Generator().manual_seed(2)).to(dev)
    monkeypatch.setattr(M, "SHARED_MIN_TOKENS", 0)
    for least in (0, 1 << 60):
        monkeypatch.setattr(M, "SHARED_MIN_BYTES", least)
        tokens, found = model.generate(ids, max_length=12, do_sample=False, eos_token_id=None, num_samples=3,
                                       return_logprobs=True, top_logprobs=3, use_graph=use_graph)
        assert tokens.shape == (6, 62) and found.logprobs.shape == (6, 12) and found.top_tokens.shape == (6, 12, 3)
        assert torch.equal(tokens, tokens[::3].repeat_interleave(3, dim=0))
        assert torch.equal(found.top_tokens[..., 0], tokens[:, 50:])
        with torch.no_grad():
            again = model.score(tokens, top_k=3)
        assert (again.logprobs[:, 49:] - found.logprobs).abs().max() <= 0.05
        assert (again.entropy[:, 49:] - found.entropy).abs().max() <= 0.05


def test_generate_draws_differ(M, dev):
    model = model_of(M, dev)
    ids = torch.randint(0, 512, (1, 40), generator=torch.Generator().manual_seed(3)).to(dev)
    out = model.generate(ids, max_length=16, eos_token_id=None, num_samples=8, temperature=2.0, top_p=1.0)
    assert out.shape == (8, 56) and len({tuple(r.tolist()) for r in out}) > 1


def test_score_gradient(M, dev):
    """Through the torch backend's logits, against autograd of log_softmax, in fp32."""
    model = model_of(M, dev, dtype=torch.float32, attn_impl="torch")
    ids = torch.randint(0, 512, (2, 20), generator=torch.Generator().manual_seed(4)).to(dev)
    r = model.score(ids)
    (r.logprobs.sum() + 0.1 * r.entropy.sum()).backward()
    got = model.token_embedding.weight.grad.clone()
    model.zero_grad()
    logp = torch.log_softmax(model(ids)["logits"], dim=-1)[:, :-1]
    (logp.gather(2, ids[:, 1:, None]).sum() - 0.1 * (logp.exp() * logp).sum()).backward()
    ref = model.token_embedding.weight.grad
    assert (got - ref).abs().max() <= 1e-4 * ref.abs().max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cached", [False, True])
def test_non_causal_attention(M, dev, dtype, cached):
    """config.causal False at inference runs over the pages; under autograd in torch: the same
    attention."""
    model = model_of(M, dev, dtype=dtype, causal=False)
    attn = model.blocks[0].attention
    x = (torch.randn(2, 70, 256, generator=torch.Generator().manual_seed(5)) * 0.5).to(dev, dtype)

    def both():
        cache = model.new_kv_cache(2, 70) if cached else None
        if not cached:
            return attn(x)[0]
        cache.num_layers, outs = 1, []
        for part in (x[:, :33], x[:, 33:34], x[:, 34:]):
            outs.append(attn(part, kv_cache=cache)[0])
        return torch.cat(outs, dim=1)

    with torch.no_grad():
        got = both()
    ref = both().detach()  # (gradients on: the torch evaluation)
    assert (got.float() - ref.float()).abs().max() <= {torch.float16: 2e-3, torch.bfloat16: 1.6e-2}[dtype]


@pytest.mark.parametrize("kw", [{"d_model": 128}, {"kv_block_size": 32}, {"d_model": 128, "kv_block_size": 8}], ids=str)
def test_non_causal_attention_of_other_geometries(M, dev, kw):
    """Head dims and page sizes that the kernel does not take: through torch, with a cache and
    without, as under autograd."""
    model = model_of(M, dev, dtype=torch.float16, causal=False, **kw)
    attn = model.blocks[0].attention
    width = kw.get("d_model", 256)
    x = (torch.randn(2, 21, width, generator=torch.Generator().manual_seed(6)) * 0.5).to(dev, torch.float16)

    def both():
        cache = model.new_kv_cache(2, 21)
        cache.num_layers = 1
        return torch.cat([attn(x[:, :13], kv_cache=cache)[0], attn(x[:, 13:], kv_cache=cache)[0], attn(x)[0]], dim=1)

    with torch.no_grad():
        got = both()
    assert (got.float() - both().detach().float()).abs().max() <= 2e-3
