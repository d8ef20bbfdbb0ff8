"""Token log probabilities, entropy, top tokens and their gradient on the GPU vs float64.

Tolerances.  Forward, fp32 arithmetic on the logits as given: z - m is exact or off by 2^-24 |z - m|,
exponentials and their sums by a few 2^-24 relative: 16 * 2^-24 of (1 + |logp|) covers the sum's log,
and the entropy, a sum of weights that are each so far off, the same of (1 + H).  Gradient: p, logp
and the sum of the upstream gradients each to 2^-21 of themselves, then half a step of the output
type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged_kv as orc

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def to64(t):
    return t.detach().double().cpu().numpy()


def make(n, v, dtype, seed, pad=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    z = (torch.randn(n, v + pad, generator=gen) * spread).to(dtype)[:, :v]
    t = torch.randint(0, v, (n,), generator=gen)
    t[n // 2:n // 2 + 1] = -100
    return z, t


def compare(r, z, t, k, what=""):
    lp, h, top, ids = orc.token_logprobs(to64(z), t.numpy(), k)
    for got, ref, name in ((r.logprobs, lp, "logprobs"), (r.entropy, h, "entropy"), (r.top_logprobs, top, "top")):
        got = to64(got)
        assert got.shape == ref.shape, (what, name)
        same = (np.isnan(got) & np.isnan(ref)) | (got == ref)
        with np.errstate(invalid="ignore"):
            near = np.abs(got - ref) <= 16 * 2.0 ** -24 * (1 + np.abs(ref))
        assert (same | near).all(), f"{what} {name}: {got[~(same | near)][:4]} against {ref[~(same | near)][:4]}"
    assert np.array_equal(r.top_tokens.cpu().numpy(), ids), f"{what}: top tokens"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 7, 7), (5, 64, 3), (2, 100, 64), (4, 511, 20), (3, 4097, 33),
                                   (2, 32000, 20), (300, 777, 5), (1, 131072, 64), (2, 50257, 0)])
@pytest.mark.parametrize("pad", [0, 3])
def test_logprobs_vs_oracle(iva, dev, dtype, n, v, k, pad):
    """Vocabularies from one to many tokens, odd sizes, rows that start anywhere within 16 bytes."""
    z, t = make(n, v, dtype, n * v + k, pad)
    compare(iva.token_logprobs(z.to(dev) if not pad else torch.nn.functional.pad(z, (0, pad)).to(dev)[:, :v],
                               t.to(dev), k), z, t, k, f"{n}x{v} top {k}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few values", "large offset", "peaked"])
def test_logprobs_orders_and_ties(iva, dev, dtype, kind):
    """Equal logits go by index; sorted rows insert at every step; a common offset costs nothing;
    a row of one likely token has an entropy near zero."""
    v, k = 5003, 40
    i = torch.arange(v, dtype=torch.float64)
    row = {"equal": i * 0 + 1.5, "rising": i / 256, "falling": -i / 256, "few values": (i * 7919 % 5),
           "large offset": 30000 + (i * 7919 % 97) / 4, "peaked": torch.where(i == 4711, 60.0, 0.0)}[kind]
    z = torch.stack([row, row.flip(0)]).to(dtype)
    t = torch.tensor([4711, 3])
    compare(iva.token_logprobs(z.to(dev), t.to(dev), k), z, t, k, kind)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_logprobs_masked_and_not_finite(iva, dev, dtype):
    """-inf and lowest-value masks, rows of only masks, NaN and +inf, by row."""
    v, k = 3001, 6
    z, t = make(9, v, dtype, 5)
    low = torch.finfo(dtype).min
    z[0, 10:] = float("-inf")
    z[1, 3:] = float("-inf")               # fewer candidates than tops
    z[2] = float("-inf")
    z[3, 100:] = low
    z[4] = low
    z[5, 17] = float("nan")
    z[6, 18] = float("inf")
    z[7, 18:20] = float("inf")
    z[8, ::2] = float("-inf")
    t[:5] = torch.tensor([4, 2000, 1, 50, 7])
    t[8] = 2                                # a masked token: -inf
    r = iva.token_logprobs(z.to(dev), t.to(dev), k)
    compare(r, z, t, k, "masks")
    assert torch.isneginf(r.logprobs[[1, 2, 8]]).all() and (r.entropy[2] == 0)
    assert r.top_tokens[5, 0] == 17 and r.top_tokens[6, 0] == 18


def grad_ref(z, t, ids, g, gh, gt):
    """The formula in float64, and the size its roundings go by."""
    z, v = to64(z), z.shape[1]
    lp_t, h, _, _ = orc.token_logprobs(z, t.numpy(), 0)
    d = z - z.max(axis=1, keepdims=True)
    logp = d - np.log(np.exp(d).sum(axis=1, keepdims=True))
    p = np.exp(logp)
    given = ((t >= 0) & (t < v)).numpy()
    g = np.where(given, g, 0.0)
    out = -p * ((g + gt.sum(axis=1))[:, None] + gh[:, None] * (np.where(p > 0, logp, 0) + h[:, None]))
    size = p * ((np.abs(g) + np.abs(gt).sum(axis=1))[:, None] + np.abs(gh)[:, None] * (np.where(p > 0, -logp, 0) + h[:, None]))
    for i in range(len(z)):
        if given[i]:
            out[i, t[i]] += g[i]
            size[i, t[i]] += abs(g[i])
        for j, x in zip(ids[i], gt[i]):
            out[i, j] += x
            size[i, j] += abs(x)
    return out, size


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k,pad", [(1, 1, 1, 0), (4, 511, 0, 0), (6, 3000, 5, 0), (3, 4099, 64, 5), (40, 257, 2, 0)])
def test_logprobs_gradient(iva, dev, dtype, n, v, k, pad):
    """Through log probabilities, entropy and tops, equal tops and tokens among them; padding tokens
    pass nothing; the input's own gradient shape and type."""
    z, t = make(n, v, dtype, 77 + v, pad)
    gen = torch.Generator().manual_seed(1)
    g, gh, gt = torch.randn(n, generator=gen), torch.randn(n, generator=gen), torch.randn(n, k, generator=gen)
    leaf = torch.nn.functional.pad(z, (0, pad)).to(dev).requires_grad_()
    r = iva.token_logprobs(leaf[:, :v], t.to(dev), k)
    torch.autograd.backward((r.logprobs, r.entropy, r.top_logprobs), [x.to(dev) for x in (g, gh, gt)])
    got = to64(leaf.grad)
    assert leaf.grad.dtype == dtype and not got[:, v:].any()
    ref, size = grad_ref(z, t, r.top_tokens.cpu().numpy(), *(x.double().numpy() for x in (g, gh, gt)))
    bound = 2.0 ** -21 * 4 * size + HALF_STEP[dtype] * np.abs(ref) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = np.abs(got[:, :v] - ref)
    assert (err <= bound).all(), f"{float((err - bound).max()):.3e} past the bound"


def test_logprobs_gradient_against_differences(iva, dev):
    """Central differences of the oracle's float64 values along random directions."""
    z, t = make(3, 200, torch.float32, 9, spread=1.0)
    leaf = z.to(dev).requires_grad_()
    r = iva.token_logprobs(leaf, t.to(dev), 4)
    (r.logprobs.sum() + 0.3 * r.entropy.sum() + (r.top_logprobs * torch.arange(4, device=dev)).sum()).backward()
    grad = to64(leaf.grad)
    rng = np.random.default_rng(0)

    def value(x):
        lp, h, top, _ = orc.token_logprobs(x, t.numpy(), 4)
        return lp.sum() + 0.3 * h.sum() + (top * np.arange(4)).sum()

    for _ in range(5):
        u = rng.standard_normal(z.shape)
        eps = 1e-6
        num = (value(to64(z) + eps * u) - value(to64(z) - eps * u)) / (2 * eps)
        assert abs((grad * u).sum() - num) <= 1e-4 * (1 + abs(num))


def test_logprobs_gradient_of_masked_rows(iva, dev):
    z, t = make(3, 300, torch.bfloat16, 6)
    z[0] = float("-inf")
    z[1, ::3] = float("-inf")
    t[:] = torch.tensor([4, 3, 8])
    leaf = z.to(dev).requires_grad_()
    r = iva.token_logprobs(leaf, t.to(dev), 2)
    (r.logprobs[2] + r.entropy.sum()).backward()
    assert torch.isfinite(leaf.grad).all() and not leaf.grad[0].any() and not leaf.grad[1, ::3].any()


def test_logprobs_shapes_and_modes(iva, dev):
    """Leading dims, no rows, strided and expanded rows, int32 tokens, no graph without grad."""
    z, t = make(6, 130, torch.float16, 8)
    zd, td = z.to(dev), t.to(dev)
    r = iva.token_logprobs(zd.view(2, 3, 130), td.view(2, 3).int(), 3)
    assert r.logprobs.shape == (2, 3) and r.top_tokens.shape == (2, 3, 3)
    flat = iva.token_logprobs(zd, td, 3)
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(r, flat))
    turned = iva.token_logprobs(zd.t().contiguous().t(), td, 3)
    assert all(torch.equal(a, b) for a, b in zip(turned, flat))
    same = iva.token_logprobs(zd[:1].expand(6, 130), td, 3)
    assert torch.equal(same.entropy, flat.entropy[:1].expand(6))
    one = iva.token_logprobs(zd[2], td[2], 3)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, flat.top_tokens[2])
    none = iva.token_logprobs(zd[:0], td[:0], 3)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 3)
    leaf = zd.clone().requires_grad_()
    with torch.no_grad():
        assert not iva.token_logprobs(leaf, td).logprobs.requires_grad
    empty = iva.token_logprobs(leaf[:0], td[:0])
    assert torch.autograd.grad(empty.logprobs.sum(), leaf)[0].abs().sum() == 0
    with pytest.raises(RuntimeError):  # once differentiable
        g, = torch.autograd.grad(iva.token_logprobs(leaf, td).logprobs.sum(), leaf, create_graph=True)
        g.sum().backward()


def test_logprobs_graph(iva, dev):
    """Forward and backward captured and replayed on new logits, beside eager calls."""
    z, t = make(5, 1000, torch.float32, 10)
    leaf, td = z.to(dev).requires_grad_(), t.to(dev)

    def both():
        r = iva.token_logprobs(leaf, td, 4)
        return (*(x.detach() for x in r), torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)[0])

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        both()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs = both()
    for step in range(3):
        with torch.no_grad():
            leaf.copy_(torch.randn(z.shape, generator=torch.Generator().manual_seed(step)))
        want = [x.clone() for x in both()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), step
