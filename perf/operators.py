"""Three operators of a serving and scoring program, in their plain form and through the
package: what they are measured on.

Kinds of cases (field ``kind``):
  prefix  one decode step's attention of a batch whose sequences share their prompts' pages:
          groups of rows with one prefix each, a suffix of its own per row
  cross   attention of a decoder's rows to an encoder's states of another length, kept in pages
  logp    log probabilities of given tokens, entropy and the k most likely tokens of rows of
          logits, or, with ``grad``, the first two and the gradient of the logits

The pools hold pages of 16 tokens, K as [page, head, dim / X, token, X] with X = 16 bytes of
elements, V as [page, head, dim, token]; FP8 pages hold e4m3 codes, value = code / factor, V in the
order [dim % 16, token / 4, dim / 16, token % 4].
"""
from __future__ import annotations

import math
import random

import torch

own = False

BS = 16
FP8 = torch.float8_e4m3fn
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------- cases

def listed():
    return [
        # Two answers to one short prompt: the smallest use, where latency counts.
        dict(name="prefix-2", kind="prefix", dtype="bf16", pages="bf16", groups=1, least=2, most=2, prefix_lo=512,
             prefix_hi=512, own_lo=3, own_hi=40, hq=32, hkv=8, dim=128, window=0, sinks=0),
        # Sixteen samples of one long prompt, some way into their answers.
        dict(name="prefix-16", kind="prefix", dtype="fp16", pages="fp16", groups=1, least=16, most=16,
             prefix_lo=8192, prefix_hi=8192, own_lo=1, own_hi=512, hq=32, hkv=8, dim=128, window=0, sinks=0),
        # A serving batch behind one system prompt of 4000 tokens (its last page is not full), FP8 pages.
        dict(name="prefix-64-fp8", kind="prefix", dtype="bf16", pages="fp8", groups=1, least=64, most=64,
             prefix_lo=4000, prefix_hi=4000, own_lo=16, own_hi=2048, hq=32, hkv=8, dim=128, window=0, sinks=0),
        # Several prompts with differing numbers of samples and lengths, as a scheduler mixes them.
        dict(name="prefix-groups", kind="prefix", dtype="bf16", pages="bf16", groups=9, least=1, most=24,
             prefix_lo=333, prefix_hi=7000, own_lo=0, own_hi=600, hq=32, hkv=8, dim=128, window=0, sinks=0),
        # A large batch on one very long shared document.
        dict(name="prefix-256", kind="prefix", dtype="fp16", pages="fp16", groups=1, least=256, most=256,
             prefix_lo=16384, prefix_hi=16384, own_lo=32, own_hi=256, hq=32, hkv=8, dim=128, window=0, sinks=0),
        # A decoder's single-token step on four encoded inputs.
        dict(name="cross-4x1", kind="cross", dtype="fp16", pages="fp16", batch=4, rows_lo=1, rows_hi=1, keys_lo=1500,
             keys_hi=1500, hq=16, hkv=16, dim=64),
        # Beams of five rows on sixteen inputs of ragged length.
        dict(name="cross-16x5", kind="cross", dtype="bf16", pages="bf16", batch=16, rows_lo=5, rows_hi=5, keys_lo=301,
             keys_hi=1500, hq=32, hkv=8, dim=128),
        # Whole target sequences at once (scoring, or a prompt of the decoder).
        dict(name="cross-16x448", kind="cross", dtype="bf16", pages="bf16", batch=16, rows_lo=97, rows_hi=448,
             keys_lo=700, keys_hi=1500, hq=16, hkv=16, dim=64),
        # A sampling step's log probabilities with the alternatives an API returns.
        dict(name="logp-4", kind="logp", dtype="bf16", rows=4, vocab=32000, top=20, grad=False, stride=0),
        # Scores of a batch of answers, top five, fp32 logits of a large vocabulary.
        dict(name="logp-512-fp32", kind="logp", dtype="fp32", rows=512, vocab=131072, top=5, grad=False, stride=0),
        # Scores of a batch of prompts: every position's token.
        dict(name="logp-8192", kind="logp", dtype="bf16", rows=8192, vocab=32000, top=0, grad=False, stride=0),
        # A policy update: log probabilities and entropy with their gradient.
        dict(name="logp-4096-grad", kind="logp", dtype="bf16", rows=4096, vocab=32000, top=0, grad=True, stride=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = [(32, 8), (32, 8), (16, 16), (8, 1), (16, 4), (12, 4), (8, 2)]


def draw(rng: random.Random):
    while True:
        kind = rng.choice(["prefix", "prefix", "cross", "logp"])
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        if kind == "logp":
            c = dict(kind=kind, dtype=dtype, rows=_log_int(rng, 1, 8192),
                     vocab=rng.choice([512, 32000, 50257, 131072, _log_int(rng, 2, 200000)]), top=0,
                     grad=rng.random() < 0.3, stride=rng.choice([0, 0, 8, 13]))
            if not c["grad"]:
                c["top"] = min(rng.choice([0, 1, 5, 20, 32]), c["vocab"])
            if c["rows"] * c["vocab"] > 8192 * 32000:
                continue
            return c
        hq, hkv = rng.choice(_HEADS)
        c = dict(kind=kind, dtype=dtype, pages=dtype, hq=hq, hkv=hkv, dim=rng.choice([64, 128, 128, 256]))
        if dtype != "fp32" and rng.random() < 0.3:
            c["pages"] = "fp8"
        if kind == "prefix":
            most = _log_int(rng, 1, 64)
            hi, own_hi = _log_int(rng, 16, 16384), _log_int(rng, 1, 2048)
            c.update(groups=_log_int(rng, 1, 16), least=rng.randint(1, most), most=most,
                     prefix_lo=_log_int(rng, 1, hi), prefix_hi=hi, own_lo=rng.randint(0, own_hi), own_hi=own_hi,
                     window=0, sinks=0)
            if rng.random() < 0.2:
                c.update(window=_log_int(rng, 64, 4096), sinks=rng.choice([0, 4]))
        else:
            hi, rows = _log_int(rng, 1, 4096), _log_int(rng, 1, 448)
            c.update(batch=_log_int(rng, 1, 32), rows_lo=rng.randint(0, rows), rows_hi=rows,
                     keys_lo=rng.randint(0, hi), keys_hi=hi)
        w = work(c)
        pool = _pool_pages(c, _groups(c)[2] if kind == "prefix" else []) * c["hkv"] * c["dim"] * 2 * BS * (4 if dtype == "fp32" else 2)
        if pool > 1 << 30 or w["bytes"] > 5e8 or w["flops"] > (6e10 if dtype != "fp32" else 1e10):
            continue
        return c


# ----------------------------------------------------------------------- geometry

def _spread(lo, hi, n):
    """n whole numbers from lo to hi, both among them, spread evenly."""
    return [hi] if n == 1 else [round(lo + (hi - lo) * i / (n - 1)) for i in range(n)]


def _groups(c):
    """(rows of each group, shared tokens of each group, each row's own tokens)."""
    sizes = _spread(c["least"], c["most"], c["groups"])
    prefixes = _spread(c["prefix_hi"], c["prefix_lo"], c["groups"])
    return sizes, prefixes, _spread(c["own_lo"], c["own_hi"], sum(sizes))


def _rows_of(c):
    """cross: (query rows, keys) of each sequence."""
    return _spread(c["rows_lo"], c["rows_hi"], c["batch"]), _spread(c["keys_hi"], c["keys_lo"], c["batch"])


def _pool_pages(c, owns):
    if c["kind"] == "cross":
        return max(1, sum(-(-n // BS) for n in _rows_of(c)[1]))
    sizes, prefixes, _ = _groups(c)
    total, at = 0, 0
    for n, p in zip(sizes, prefixes):
        total += p // BS + sum(-(-(p + o) // BS) - p // BS for o in owns[at:at + n])
        at += n
    return max(1, total)


def _layout(c, seed):
    """(lengths, block table on the host, pages) on a seeded permutation of the pool's pages; the
    rows of a group share the pages that its prefix fills, and take the own lengths in seeded order."""
    r = random.Random(seed)
    owns = [] if c["kind"] == "cross" else _groups(c)[2]
    r.shuffle(owns)
    pages = _pool_pages(c, owns)
    perm = list(range(pages))
    r.shuffle(perm)
    rows, lengths, at = [], [], 0
    if c["kind"] == "cross":
        lengths = _rows_of(c)[1]
        for n in lengths:
            rows.append(perm[at:at + -(-n // BS)])
            at += -(-n // BS)
    else:
        for n, p in zip(*_groups(c)[:2]):
            shared = perm[at:at + p // BS]
            at += p // BS
            for _ in range(n):
                length = p + owns[len(rows)]
                tail = -(-length // BS) - p // BS
                rows.append(shared + perm[at:at + tail])
                lengths.append(length)
                at += tail
    table = torch.full((len(rows), max(1, max(map(len, rows)))), -1, dtype=torch.int32)
    for b, own_pages in enumerate(rows):
        table[b, :len(own_pages)] = torch.tensor(own_pages, dtype=torch.int32)
    return lengths, table, pages


def _gen(seed, i):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + i) % (1 << 62))


def _randn(shape, seed, i, dtype):
    return torch.randn(shape, generator=_gen(seed, i), device="cuda", dtype=dtype)


def _pools(c, seed, pages):
    """K and V pools of N(0, 1) rows (and the FP8 factors)."""
    hkv, d = c["hkv"], c["dim"]
    if c["pages"] != "fp8":
        dt = DTYPES[c["pages"]]
        x = 16 // dt.itemsize
        return (_randn((pages, hkv, d // x, BS, x), seed, 1, dt), _randn((pages, hkv, d, BS), seed, 2, dt), {})
    out, scales = [], []
    for i in (1, 2):
        rows = _randn((pages, hkv, BS, d), seed, i, torch.float32)
        sf = torch.full((), 448.0, device="cuda") / rows.abs().amax(dim=-1)
        out.append((rows * sf[..., None]).to(FP8).view(torch.uint8))
        scales.append(sf.contiguous())
    k = out[0].view(pages, hkv, BS, d // 16, 16).permute(0, 1, 3, 2, 4).contiguous()
    v = out[1].view(pages, hkv, 4, 4, d // 16, 16).permute(0, 1, 5, 2, 4, 3).contiguous().view(pages, hkv, d, BS)
    return k.view(FP8), v.view(FP8), {"k_scale": scales[0], "v_scale": scales[1]}


# ------------------------------------------------------------------- prepare, run

def prepare(case, seed):
    c = case
    if c["kind"] == "logp":
        n, v, dt = c["rows"], c["vocab"], DTYPES[c["dtype"]]
        # logits of a language model: a broad bulk and some tokens well above it
        z = torch.randn((n, v + c["stride"]), generator=_gen(seed, 1), device="cuda", dtype=torch.float32)
        z = (z * 2 + z.relu().pow(3) * 0.1).to(dt)[:, :v]
        tokens = torch.randint(0, v, (n,), generator=_gen(seed, 2), device="cuda")
        tokens = torch.where(torch.arange(n, device="cuda") % 17 == 16, -100, tokens)  # padding
        s = dict(kind="logp", z=z, tokens=tokens, top=c["top"], grad=c["grad"])
        if c["grad"]:
            s.update(g=_randn((n,), seed, 3, torch.float32), gh=_randn((n,), seed, 4, torch.float32) * 0.01)
        return s
    lengths, table, pages = _layout(c, seed)
    k_pool, v_pool, kw = _pools(c, seed, pages)
    dt = DTYPES[c["dtype"]]
    s = dict(kind=c["kind"], k_pool=k_pool, v_pool=v_pool, kw=kw, tables=table.cuda(), lengths=lengths,
             lens=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if c["kind"] == "prefix":
        sizes, prefixes, _ = _groups(c)
        start = torch.tensor([0] + sizes).cumsum(0).to(torch.int32)
        s.update(q=_randn((sum(sizes), c["hq"], c["dim"]), seed, 4, dt), start=start.cuda(),
                 prefixes=torch.tensor(prefixes, dtype=torch.int32, device="cuda"), largest=max(sizes),
                 window=c["window"], sinks=c["sinks"])
    else:
        rows = _rows_of(c)[0]
        start = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
        s.update(q=_randn((sum(rows), c["hq"], c["dim"]), seed, 4, dt), start=start.cuda(), rows=rows,
                 longest=max(rows))
    return s


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "logp":
        return _logp_plain(s)
    counts = [1] * len(s["lengths"]) if s["kind"] == "prefix" else s["rows"]
    outs, at = [], 0
    for b, (n, length) in enumerate(zip(counts, s["lengths"])):
        outs.append(_attend(s, b, s["q"][at:at + n], length))
        at += n
    return [torch.cat(outs)]


def _run_own(s):
    from __graft_entry__ import load_package
    iva = load_package()
    if s["kind"] == "logp":
        if not s["grad"]:
            r = iva.token_logprobs(s["z"], s["tokens"], top_k=s["top"])
            return [r.logprobs, r.entropy] + ([r.top_logprobs, r.top_tokens] if s["top"] else [])
        z = s["z"].detach().requires_grad_()
        r = iva.token_logprobs(z, s["tokens"])
        dz, = torch.autograd.grad((r.logprobs, r.entropy), z, (s["g"], s["gh"]))
        return [r.logprobs.detach(), r.entropy.detach(), dz]
    if s["kind"] == "cross":
        return [iva.paged_cross_attention(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["lens"], s["start"],
                                          max_query_len=s["longest"], **s["kw"])]
    return [iva.paged_prefix_decode_attention(
        s["q"], s["k_pool"], s["v_pool"], s["tables"], s["lens"], s["start"], s["prefixes"], window=s["window"],
        n_sink=s["sinks"], max_group=s["largest"], **s["kw"])]


def _page_rows(s, pages):
    """K and V of whole pages as float32 [Hkv, tokens, D]."""
    k, v, kw = s["k_pool"], s["v_pool"], s["kw"]
    n, hkv, d = pages.numel(), v.shape[1], v.shape[2]
    if kw:
        kc, vc = (t.view(torch.uint8)[pages].view(FP8).float() for t in (k, v))
        vc = vc.view(n, hkv, 16, 4, d // 16, 4).permute(0, 1, 4, 2, 3, 5).reshape(n, hkv, d, BS)
        kc = kc / kw["k_scale"][pages][:, :, None, :, None]
        vc = vc / kw["v_scale"][pages][:, :, None, :]
    else:
        kc, vc = k[pages].float(), v[pages].float()
    kr = kc.permute(1, 0, 3, 2, 4).reshape(hkv, n * BS, d)
    return kr, vc.permute(1, 0, 3, 2).reshape(hkv, n * BS, d)


def _attend(s, b, q, length):
    """softmax(q k^T / sqrt(D)) v of the rows q [n, Hq, D] over sequence b's visible keys."""
    n, hq, d = q.shape
    if length == 0 or n == 0:
        return torch.zeros_like(q)
    k, v = _page_rows(s, s["tables"][b, :-(-length // BS)].long())
    k, v = k[:, :length], v[:, :length]
    hkv = k.shape[0]
    qg = q.float().view(n, hkv, hq // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
    scores = torch.matmul(qg, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
    if s.get("window"):
        pos = torch.arange(length, device=q.device)
        hidden = (pos < length - s["window"]) & (pos >= s["sinks"])
        scores = torch.where(hidden, float("-inf"), scores)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    return o.view(hkv, n, hq // hkv, d).permute(1, 0, 2, 3).reshape(n, hq, d).to(q.dtype)


def _logp_plain(s):
    parts = []
    for i in range(0, s["z"].shape[0], 1024):
        rows = slice(i, i + 1024)
        z, tokens = s["z"][rows].float(), s["tokens"][rows]
        given = (tokens >= 0) & (tokens < z.shape[1])
        t = torch.where(given, tokens, 0)[:, None]
        m = z.amax(dim=-1, keepdim=True)
        e = torch.exp(z - m)
        total = e.sum(dim=-1, keepdim=True)
        logp = z - m - torch.log(total)
        p = e / total
        entropy = -(p * logp).sum(dim=-1)
        out = [torch.where(given, logp.gather(1, t)[:, 0], 0.0), entropy]
        if s["grad"]:
            g = torch.where(given, s["g"][rows], 0.0)[:, None]
            dz = -g * p - s["gh"][rows][:, None] * p * (logp + entropy[:, None])
            out.append(dz.scatter_add_(1, t, g).to(s["z"].dtype))
        elif s["top"]:
            order = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
            out += [logp.gather(1, order), order]
        parts.append(out)
    return [torch.cat(p) for p in zip(*parts)]


# --------------------------------------------------------------------------- work

def work(case):
    """Bytes and operations that a pass cannot do without: shared pages count once."""
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "logp":
        n, v = c["rows"], c["vocab"]
        out = 8.0 * n + 12.0 * n * c["top"] + (n * v * e + 8.0 * n if c["grad"] else 0)
        return {"bytes": n * v * e + 8.0 * n + out, "flops": n * v * (10.0 if c["grad"] else 5.0)}
    row = 2 * c["hkv"] * {"fp8": c["dim"] + 4, "fp32": 4 * c["dim"]}.get(c["pages"], 2 * c["dim"])
    if c["kind"] == "cross":
        rows, keys = _rows_of(c)
        return {"bytes": float(row * sum(k for n, k in zip(rows, keys) if n) + 2 * sum(rows) * c["hq"] * c["dim"] * e
                               + 4 * sum(-(-k // BS) for k in keys)),
                "flops": 4.0 * c["hq"] * c["dim"] * sum(n * k for n, k in zip(rows, keys))}
    sizes, prefixes, owns = _groups(c)
    read, seen, at = 0, 0, 0
    for n, p in zip(sizes, prefixes):
        lengths = [p + o for o in owns[at:at + n]]
        at += n
        shared = p // BS * BS
        first = [max(0, length - c["window"]) if c["window"] else 0 for length in lengths]
        sinks = c["sinks"] if c["window"] else 0
        seen += sum(length - f + min(sinks, f) for length, f in zip(lengths, first))
        low = min(min(first), shared)
        read += shared - low + min(sinks, low)
        read += sum(max(0, length - max(shared, f)) for length, f in zip(lengths, first))
    rows = sum(sizes)
    return {"bytes": float(row * read + 2 * rows * c["hq"] * c["dim"] * e + 4 * (read // BS + 2 * rows)),
            "flops": 4.0 * c["hq"] * c["dim"] * seen}


# -------------------------------------------------------------------------- exact

@torch.no_grad()
def exact(case, seed):
    """The outputs in float64, from the definitions."""
    s = prepare(case, seed)
    if case["kind"] == "logp":
        return _logp_exact(s)
    d, hkv = case["dim"], case["hkv"]
    per = case["hq"] // hkv
    counts = [1] * len(s["lengths"]) if s["kind"] == "prefix" else s["rows"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(zip(counts, s["lengths"])):
        j = torch.arange(length, device="cuda")
        if s.get("window"):
            j = j[(j >= length - s["window"]) | (j < s["sinks"])]
        if n and j.numel():
            page, slot = s["tables"][b].long()[j // BS], j % BS
            for h in range(hkv):
                k, v = _head_rows(s, page, slot, h)
                q = s["q"][at:at + n, h * per:(h + 1) * per].double().reshape(-1, d)
                w = torch.softmax(torch.matmul(q, k.t().contiguous()) / math.sqrt(d), dim=1)
                out[at:at + n, h * per:(h + 1) * per] = torch.matmul(w, v).view(n, per, d)
        at += n
    return [out]


def _head_rows(s, page, slot, h):
    """K and V [keys, D] of one head at (page, slot), in float64, element by element."""
    k, v, kw = s["k_pool"], s["v_pool"], s["kw"]
    d = v.shape[2]
    i = torch.arange(d, device="cuda")
    x = k.shape[-1]
    flat_k = ((page * k.shape[1] + h)[:, None] * (d // x) + i // x) * BS * x + slot[:, None] * x + i % x
    tile = (page * v.shape[1] + h)[:, None] * d * BS
    if not kw:
        return k.flatten()[flat_k].double(), v.flatten()[tile + i * BS + slot[:, None]].double()
    inner = (((i % 16) * 4 + slot[:, None] // 4) * (d // 16) + i // 16) * 4 + slot[:, None] % 4
    codes = [t.view(torch.uint8).flatten()[f].view(FP8).double() for t, f in ((k, flat_k), (v, tile + inner))]
    return [x / kw[n][page, h, slot].double()[:, None] for x, n in zip(codes, ("k_scale", "v_scale"))]


def _logp_exact(s):
    outs = []
    for i in range(0, s["z"].shape[0], 512):
        z, tokens = s["z"][i:i + 512].double(), s["tokens"][i:i + 512]
        v = z.shape[1]
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        p = torch.exp(logp)
        h = -(p * logp).sum(dim=1)
        one = (torch.arange(v, device="cuda")[None, :] == tokens[:, None])
        out = [torch.where(one, logp, 0.0).sum(dim=1), h]
        if s["grad"]:
            g, gh = s["g"][i:i + 512].double()[:, None], s["gh"][i:i + 512].double()[:, None]
            out.append(torch.where(one, g, 0.0) - one.any(dim=1, keepdim=True) * g * p
                       - gh * p * (logp + h[:, None]))
        elif s["top"]:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s["top"]]
            out += [logp.gather(1, order), order]
        outs.append(out)
    return [torch.cat(p) for p in zip(*outs)]
