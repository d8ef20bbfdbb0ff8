"""Forking a cache into samples, and scoring, on the CPU: page bookkeeping, refusals, the torch
formulas."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def P(iva):
    from importlib import import_module
    return import_module("iva_amd.paged_cache")


@pytest.fixture(scope="module")
def M(iva):
    from importlib import import_module
    return import_module("iva_amd.model")


def cache_of(P, batch, tokens, **kw):
    c = P.PagedKVCache(batch, 2, 8, 0, "cpu", torch.float32, num_layers=2, max_seq_len=64, **kw)
    c.pool.extend(c.seq_ids, tokens)
    c.seq_len = tokens
    return c


def test_cache_fork_shares_pages(P):
    c = cache_of(P, 2, 37, max_seqs=6, num_pages=40)
    for t in c.pool.k_pools + c.pool.v_pools:
        t.copy_(torch.randn(t.shape))
    before = [c.pool.pages(s) for s in c.seq_ids]
    c.fork(3)
    assert c.batch_size == 6 and len(c.seq_ids) == 6 and c.seq_len == 37
    for b in range(2):
        rows = [c.pool.pages(s) for s in c.seq_ids[3 * b:3 * b + 3]]
        assert rows[0] == before[b] and all(r[:2] == rows[0][:2] for r in rows)
        assert len({r[2] for r in rows}) == 3
        for r in rows[1:]:
            for t in c.pool.k_pools + c.pool.v_pools:
                assert torch.equal(t[r[2]], t[rows[0][2]])
    s = c.shared
    assert s.group_start.tolist() == [0, 3, 6] and s.prefix_lens.tolist() == [32, 32]
    assert s.max_group == 3 and s.saved_tokens == 2 * 2 * 32
    c.free()
    assert c.pool.num_free_pages == 40


def test_more_rows_than_the_shared_op_takes_are_not_grouped(P, monkeypatch):
    monkeypatch.setattr(P, "MAX_PREFIX_ROWS", 5)
    c = cache_of(P, 2, 37, max_seqs=6, num_pages=40)
    c.fork(3)
    assert c.batch_size == 6 and c.shared is None


def test_a_decode_step_reads_shared_pages_where_that_pays(P, M):
    """By the bytes saved, the prefix, the window and the width."""
    from types import SimpleNamespace as NS
    pool = NS(num_kv_heads=8, head_dim=128, dtype=torch.bfloat16)  # 4 KiB a token
    def cache(saved, shortest):
        return NS(seq_len=3000, pool=pool, shared=P.SharedPrefix(None, None, 8, saved, shortest))
    assert M._reads_shared(cache(7 * 2048, 2048), None, 4096)
    assert not M._reads_shared(cache(7 * 2048 - 1, 2048), None, 4096)
    assert not M._reads_shared(cache(31 * 512, 512), None, 4096)
    assert not M._reads_shared(cache(7 * 2048, 2048), 3000, 4096)
    assert M._reads_shared(cache(7 * 2048, 2048), 3001, 4096)
    assert M._reads_shared(cache(16 * 7 * 2048, 2048), None, 1024)
    assert not M._reads_shared(NS(seq_len=3000, pool=pool, shared=None), None, 4096)
    assert not M._reads_shared(None, None, 4096)


def test_cache_fork_of_a_short_or_whole_prompt(P):
    short = cache_of(P, 1, 9, max_seqs=4, num_pages=8)
    short.fork(4)
    assert short.shared is None and short.batch_size == 4  # no full page: nothing is shared
    whole = cache_of(P, 1, 32, max_seqs=2, num_pages=2)
    whole.fork(2)  # no partial page: no page is needed
    assert whole.shared.prefix_lens.tolist() == [32] and whole.pool.num_free_pages == 0
    assert whole.shared.shortest == 32
    one = cache_of(P, 1, 20)
    one.fork(1)
    assert one.shared is None and one.batch_size == 1


def test_cache_fork_refusals_change_nothing(P):
    c = cache_of(P, 2, 20, max_seqs=4, num_pages=5)
    state = c.pool.state_dict()
    with pytest.raises(P.OutOfPagesError, match="pages"):
        c.fork(2)                      # two partial pages, one left
    with pytest.raises(P.OutOfPagesError, match="rows"):
        cache_of(P, 2, 20, num_pages=40).fork(2)
    with pytest.raises(ValueError, match="samples"):
        c.fork(0)
    after = c.pool.state_dict()
    assert all(str(state[k]) == str(after[k]) for k in state) and c.batch_size == 2
    c._cursor = 1
    with pytest.raises(RuntimeError, match="forward"):
        c.fork(2)


def test_fork_many_refusals(P):
    pool = P.PagedKVPool(8, 1, 8, device="cpu", max_seqs=4, dtype=torch.float32)
    pool.add_sequence("a")
    pool.allocate("a", 20)
    for src, dst, error in ((["a"], ["b", "c"], ValueError), (["a", "a"], ["b", "b"], ValueError),
                            (["a"], ["a"], ValueError), (["x"], ["b"], KeyError),
                            (["a"] * 4, list("bcde"), P.OutOfPagesError)):
        with pytest.raises(error):
            pool.fork_many(src, dst)
        assert not any(pool.has_sequence(s) for s in "bcde") and pool.num_free_pages == 6


def test_update_below_a_shared_prefix_is_refused(P):
    c = cache_of(P, 1, 40, max_seqs=2, num_pages=16)
    c.fork(2)
    rows = torch.zeros(2, 2, 1, 8)
    with pytest.raises(ValueError, match="share"):
        c.update(rows, rows, 31)


def test_score_and_samples_on_the_cpu(M):
    torch.manual_seed(3)
    cfg = M.TransformerConfig(d_model=32, n_layers=1, n_heads=2, vocab_size=40, seq_len=64, dropout=0.0)
    model = M.Transformer(cfg).eval()
    ids = torch.randint(0, 40, (3, 12))
    r = model.score(ids, top_k=4)
    logp = torch.log_softmax(model(ids)["logits"], dim=-1)[:, :-1]
    assert torch.allclose(r.logprobs, logp.gather(2, ids[:, 1:, None])[..., 0], atol=1e-5)
    assert torch.allclose(r.entropy, -(logp.exp() * logp).sum(-1), atol=1e-5)
    assert r.top_tokens.shape == (3, 11, 4) and torch.allclose(r.top_logprobs, logp.gather(2, r.top_tokens), atol=1e-5)
    r.logprobs.sum().backward()
    assert model.token_embedding.weight.grad.abs().sum() > 0
    tokens, found = model.generate(ids, max_length=5, do_sample=False, eos_token_id=None, num_samples=2,
                                   return_logprobs=True, top_logprobs=2)
    plain = model.generate(ids, max_length=5, do_sample=False, eos_token_id=None)
    assert torch.equal(tokens, plain.repeat_interleave(2, dim=0))
    assert found.logprobs.shape == (6, 5) and torch.equal(found.top_tokens[..., 0], tokens[:, 12:])
    assert torch.allclose(found.logprobs, found.top_logprobs[..., 0])
    with pytest.raises(ValueError, match="num_samples"):
        model.generate(ids, num_samples=0)


def test_samples_need_a_cache_that_forks(M):
    cfg = M.TransformerConfig(d_model=32, n_layers=1, n_heads=2, vocab_size=40, seq_len=64, dropout=0.0)
    model = M.Transformer(cfg).eval()

    class Cache:  # (refused before the prompt runs through it)
        seq_len = 0

    with pytest.raises(ValueError, match="forked"):
        model.generate(torch.zeros(1, 4, dtype=torch.long), max_length=3, num_samples=2, kv_cache=Cache())


def test_logprobs_formula_masks(M):
    z = torch.tensor([[0.0, float("-inf"), 1.0], [2.0, 2.0, 2.0]])
    r = M._logprobs_of(z, torch.tensor([2, -100]), 2)
    assert torch.isfinite(r.entropy).all() and r.logprobs[1] == 0
    assert r.top_tokens.tolist() == [[2, 0], [0, 1]]
