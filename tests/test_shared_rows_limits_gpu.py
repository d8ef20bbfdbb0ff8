"""Cross attention, shared-prefix attention and token log probabilities at the ends of what they
take: pools and logits past 2^31 elements, several threads on streams of their own.  The same
content under other page ids, as a slice, or alone has to give the same bits."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

HKV, G, D = 8, 4, 128
FP8 = torch.float8_e4m3fn


def both_pools(iva, dev, dtype, n, seed=0):
    """n random pages under ids past 2^32 bytes of a large pool, and under 0 .. n - 1 of a compact
    one: [(ids, (k, v), scales), ...]."""
    gen = torch.Generator().manual_seed(seed)
    size = 1 if dtype == FP8 else 2
    edge = (1 << 32) // (HKV * D * 16 * size)  # the page whose bytes start at 2^32
    large = edge - n // 4 + torch.randperm(2 * n, generator=gen)[:n]
    k, v = ((torch.randn(n, HKV * D * 16, generator=gen)).to(dtype).to(dev) for _ in range(2))
    factors = [torch.rand(n, HKV, 16, generator=gen).to(dev) + 0.5 for _ in range(2)]
    out = []
    for ids, pages in ((large, edge + 2 * n), (torch.arange(n), n)):
        on = ids.to(dev)
        pools, scales = [], {}
        for x, shape in zip((k, v), iva.pool_shapes(pages, HKV, D, 16, dtype)):
            pool = torch.empty(shape, dtype=dtype, device=dev)
            raw = (lambda t: t.view(torch.uint8)) if dtype == FP8 else (lambda t: t)
            raw(pool).view(pages, -1)[on] = raw(x)
            pools.append(pool)
        if dtype == FP8:
            for name, f in zip(("k_scale", "v_scale"), factors):
                scales[name] = torch.empty(iva.scale_shape(pages, HKV, 16), device=dev)
                scales[name].view(pages, HKV, 16)[on] = f
        out.append((ids.to(torch.int32), pools, scales))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8], ids=str)
def test_row_attention_in_a_large_pool(iva, dev, dtype):
    keys, rows = [333, 0, 1000, 77], [1, 3, 40, 9]
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(sum(rows), HKV * G, D, generator=gen).to(dev, torch.bfloat16)
    start = torch.tensor([0] + rows).cumsum(0).int().to(dev)
    ctx = torch.tensor(keys, dtype=torch.int32, device=dev)
    need = [-(-k // 16) for k in keys]
    # one group of 64 rows on 1280 shared pages (20480 tokens) and a page of their own: 256 rows per
    # kv head, which bf16 pages walk through LDS
    shared, own = 1280, 64
    qd = torch.randn(own, HKV * G, D, generator=gen).to(dev, torch.bfloat16)
    lens = torch.randint(shared * 16 + 1, shared * 16 + 17, (own,), generator=gen).int().to(dev)
    outs = []
    for ids, pools, scales in both_pools(iva, dev, dtype, shared + own):
        bt = torch.full((len(keys), max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            bt[b, :n] = ids[at:at + n]
            at += n
        table = torch.cat([ids[:shared].expand(own, shared), ids[shared:, None]], dim=1).contiguous().to(dev)
        one = torch.tensor([0, own], dtype=torch.int32, device=dev)
        prefix = torch.tensor([shared * 16], dtype=torch.int32, device=dev)
        outs.append((iva.paged_cross_attention(q, *pools, bt.to(dev), ctx, start, max_query_len=40, **scales),
                     iva.paged_prefix_decode_attention(qd, *pools, table, lens, one, prefix, max_group=own, **scales),
                     iva.paged_decode_attention(qd, *pools, table, lens, **scales)))
        del pools
    for large, compact in zip(*outs):
        assert torch.equal(large, compact) and torch.isfinite(large).all()
    # two operators on the same rows: FP8 weights as bf16 pairs, so P's and the result's bf16 roundings
    # (2^-8 each, of values below the largest |v|, 6 factors of normal draws over 0.5) bound both
    assert (outs[0][1].float() - outs[0][2].float()).abs().max() <= 3 * 2.0 ** -8 * 12
    assert outs[0][0][1:4].abs().sum() == 0  # the sequence without keys


def test_logprobs_past_2_31_elements(iva, dev):
    n, v = (1 << 31) // 32000 + 8, 32000
    z = torch.zeros(n, v, dtype=torch.float16, device=dev)
    z[-5:] = torch.randn(5, v, generator=torch.Generator().manual_seed(2)).to(dev, torch.float16)
    t = torch.arange(n, device=dev) % v
    z.requires_grad_()
    r = iva.token_logprobs(z, t, 3)
    small = z.detach()[-5:].clone().requires_grad_()
    want = iva.token_logprobs(small, t[-5:], 3)
    assert (r.logprobs[:-5] + torch.log(torch.tensor(float(v)))).abs().max() <= 1e-5
    assert torch.equal(r.top_tokens[-5:], want.top_tokens)
    # (five rows get other numbers of waves than many: sums of 32000 fp32 terms in another order)
    for a, b in zip(r, want):
        if a.is_floating_point():
            assert (a[-5:] - b).abs().max() <= 1e-4
    g, = torch.autograd.grad((r.logprobs + 0.1 * r.entropy).sum(), z)
    gs, = torch.autograd.grad((want.logprobs + 0.1 * want.entropy).sum(), small)
    assert (g[-5:].float() - gs.float()).abs().max() <= 2.0 ** -10 and torch.isfinite(g[-5:]).all()
    assert (g[:-5].float().sum(dim=1)).abs().max() <= 32000 * 2.0 ** -25 + 2.0 ** -11


def test_logprobs_have_no_forward_gradient(iva, dev):
    """A tangent is refused, not dropped; without one the call is as ever, also without grad."""
    import torch.autograd.forward_ad as fwAD
    z = torch.randn(3, 40, generator=torch.Generator().manual_seed(3)).to(dev)
    t = torch.arange(3, device=dev)
    want = iva.token_logprobs(z, t, 2)
    with torch.no_grad(), fwAD.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(iva.token_logprobs(z, t, 2), want))
        with pytest.raises(RuntimeError):
            iva.token_logprobs(fwAD.make_dual(z, torch.ones_like(z)), t)
    graded = iva.token_logprobs(z.clone().requires_grad_(), t, 2)
    assert all(torch.equal(a, b) for a, b in zip(graded, want))
    assert graded.logprobs.requires_grad and not graded.top_tokens.requires_grad and not want.logprobs.requires_grad


def test_logprobs_capture_beside_a_live_eager_graph(iva, dev):
    """Refused while the eager results of the same leaf live; once they are dropped, captured,
    replayed and right."""
    leaf = torch.randn(4, 50, generator=torch.Generator().manual_seed(5)).to(dev).requires_grad_()
    t, other = torch.arange(4, device=dev), torch.zeros(8, device=dev)
    eager = iva.token_logprobs(leaf, t, 2)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        other.add_(1)
        with pytest.raises(RuntimeError, match="eager graph"):
            iva.token_logprobs(leaf, t, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert other.sum() == 8
    want = torch.autograd.grad((eager.logprobs + eager.entropy).sum(), leaf)[0]  # (the eager graph still works)
    del eager
    torch.cuda.synchronize()

    def both():
        r = iva.token_logprobs(leaf, t, 2)
        return torch.autograd.grad((r.logprobs + r.entropy).sum(), leaf)[0]

    with torch.cuda.stream(stream):
        both()
        again = torch.cuda.CUDAGraph()
        with torch.cuda.graph(again, stream=stream):
            got = both()
    for _ in range(2):
        got.zero_()
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_calls_from_threads_on_their_own_streams(iva, dev):
    """Each thread's workspace is its stream's: as called alone, bit for bit."""
    def inputs(seed):
        gen = torch.Generator().manual_seed(seed)
        pages, b, shared = 200, 6 + seed, 20 + 7 * seed
        ks, vs = iva.pool_shapes(pages, 2, 64, 16, torch.float16)
        pools = [torch.randn(s, generator=gen).to(dev, torch.float16) for s in (ks, vs)]
        perm = torch.randperm(pages, generator=gen).int()
        bt = torch.cat([perm[:shared].expand(b, shared), perm[shared:shared + 3 * b].view(b, 3)], dim=1)
        lens = torch.randint(shared * 16, (shared + 3) * 16, (b,), generator=gen).int()
        q = torch.randn(b, 8, 64, generator=gen).to(dev, torch.float16)
        z = torch.randn(b, 3001, generator=gen).to(dev)
        i32 = dict(dtype=torch.int32, device=dev)
        return (q, *pools, bt.contiguous().to(dev), lens.to(dev), torch.tensor([0, b], **i32),
                torch.tensor([shared * 16], **i32)), z, torch.arange(b, device=dev)

    def calls(x, n):
        args, z, t = x
        outs = []
        for _ in range(n):
            outs = [iva.paged_prefix_decode_attention(*args, max_group=args[0].shape[0]),
                    iva.paged_cross_attention(*args[:5], torch.arange(args[0].shape[0] + 1, dtype=torch.int32,
                                                                      device=dev), max_query_len=1),
                    *iva.token_logprobs(z, t, 5)]
        return outs

    data = [inputs(s) for s in range(3)]
    want = [calls(x, 1) for x in data]
    torch.cuda.synchronize()
    got = [None] * 3

    def work(i):
        s = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(s):
            got[i] = calls(data[i], 30)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("starts,prefixes,most", [([0], [], 0), ([2, 2], [64], 0), ([0, 5], [0], 5), ([1, 3, 3, 5], [64, 48, 64], 1)],
                         ids=["no-groups", "empty-group", "empty-prefix", "past-max-group"])
def test_rows_of_no_shared_walk(iva, dev, starts, prefixes, most):
    """Rows of no group, of a group without a prefix, and past max_group read all of their pages
    themselves: plain decode attention (fp16: the results' and P's half steps of values below 6,
    twice)."""
    gen = torch.Generator().manual_seed(4)
    ks, vs = iva.pool_shapes(40, 2, 64, 16, torch.float16)
    pools = [torch.randn(s, generator=gen).to(dev, torch.float16) for s in (ks, vs)]
    bt = torch.cat([torch.arange(4).expand(5, 4), 4 + torch.arange(15).view(5, 3)], dim=1).int().contiguous().to(dev)
    lens = torch.tensor([65, 112, 80, 64, 99], dtype=torch.int32, device=dev)
    q = torch.randn(5, 8, 64, generator=gen).to(dev, torch.float16)
    got = iva.paged_prefix_decode_attention(q, *pools, bt, lens, torch.tensor(starts, dtype=torch.int32, device=dev),
                                            torch.tensor(prefixes, dtype=torch.int32, device=dev), max_group=most)
    want = iva.paged_decode_attention(q, *pools, bt, lens)
    assert (got.float() - want.float()).abs().max() <= 2 * 2 * 2.0 ** -11 * 6
