"""Cross attention and decode attention behind shared prefixes on the GPU vs the fp64 oracle.

Tolerance: the weights are rounded to the pages' type before the PV product (relative u = 2^-8
bf16, 2^-11 fp16) and normalized by the sum of the rounded weights, so an output is off by at
most u max_j |v_j - o| <= 2 u max|v|; the output's own rounding adds u |o|.  FP8 pages keep weights to
16 bits (2^-16 taken).  fp32 arithmetic (scores, exponentials, sums) is given 1e-5 max|v|, the
bound of the other attention tests at unit scale.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged_kv as orc

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def to_np(t):
    return t.detach().float().cpu().numpy()


class Case:
    """Pools of random pages with NaN wherever no token lies, tables and lengths.  rows: per sequence
    (list of shared page ids, own tokens after them, length) is made by the callers below."""

    def __init__(self, iva, pages, hkv, d, dtype, fp8=False, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.gen, self.fp8, self.dtype, self.hkv, self.d = gen, fp8, dtype, hkv, d
        self.pages = pages + 2
        self.perm = (torch.randperm(pages, generator=gen) + 1).tolist()  # page 0 and the last hold NaN
        self.used = torch.zeros(self.pages, 16, dtype=torch.bool)
        self.rows = [torch.randn(self.pages, hkv, 16, d, generator=gen) for _ in range(2)]

    def take(self, tokens):
        """Pages for `tokens` tokens."""
        out = [self.perm.pop() for _ in range(-(-tokens // 16))]
        for i, p in enumerate(out):
            self.used[p, :max(0, min(16, tokens - 16 * i))] = True
        return out

    def finish(self, iva, dev):
        ks, vs = iva.pool_shapes(self.pages, self.hkv, self.d, 16, FP8 if self.fp8 else self.dtype)
        hole = ~self.used[:, None, :, None]
        k, v = self.rows
        if self.fp8:
            self.scales = []
            packed = []
            for x in (k, v):
                x = x.numpy()
                codes, sf = orc.quantize_rows(x.reshape(-1, 1, self.d))
                codes, sf = codes.reshape(x.shape).copy(), sf.reshape(x.shape[:-1]).copy()
                h = np.broadcast_to(hole.numpy()[..., 0], sf.shape)
                codes[h], sf[h] = 0x7F, np.nan  # NaN codes and factors
                packed.append(codes)
                self.scales.append(sf.astype(np.float32))
            kp = packed[0].reshape(self.pages, self.hkv, 16, self.d // 16, 16).transpose(0, 1, 3, 2, 4)
            vp = orc.fp8_v_to_tiles(np.ascontiguousarray(packed[1].transpose(0, 1, 3, 2)))
            self.np_pools = orc.dequantize_pools(np.ascontiguousarray(kp), vp, *self.scales)
            self.pools = [torch.from_numpy(np.ascontiguousarray(kp)).to(dev).view(FP8).view(ks),
                          torch.from_numpy(vp).to(dev).view(FP8).view(vs)]
            self.kw = dict(k_scale=torch.from_numpy(self.scales[0]).to(dev),
                           v_scale=torch.from_numpy(self.scales[1]).to(dev))
            return self
        nan = torch.full((), float("nan"))
        k, v = (torch.where(hole, nan, x).to(self.dtype) for x in (k, v))
        x = 16 // self.dtype.itemsize
        kp = k.view(self.pages, self.hkv, 16, self.d // x, x).permute(0, 1, 3, 2, 4).contiguous()
        vp = v.transpose(2, 3).contiguous()
        self.np_pools = (to_np(kp), to_np(vp))
        self.pools, self.kw = [kp.to(dev), vp.to(dev)], {}
        return self

    def table(self, rows, width=None):
        width = width or max(1, max(len(r) for r in rows))
        t = torch.full((len(rows), width), -1, dtype=torch.int32)
        for b, r in enumerate(rows):
            t[b, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return t

    def check(self, out, ref, what=""):
        u = HALF_STEP[self.dtype]
        vmax = float(np.nanmax(np.abs(self.np_pools[1])))
        weights = 2.0 ** -16 if self.fp8 else 0.0 if self.dtype == torch.float32 else u
        bound = (2 * weights + 1e-5) * vmax + u * np.abs(ref)
        err = np.abs(to_np(out) - ref)
        assert np.isfinite(to_np(out)).all(), f"{what}: not finite"
        assert (err <= bound).all(), f"{what}: {float((err - bound).max()):.3e} past the bound, error {err.max():.3e}"


def cross_case(iva, dev, rows, keys, hq, hkv, d, dtype, fp8=False, seed=0, holes=()):
    c = Case(iva, sum(-(-k // 16) for k in keys), hkv, d, dtype, fp8, seed)
    tables = [c.take(k) for k in keys]
    for b, j in holes:  # entries outside the pool: keys that are not attended
        tables[b][j] = -1 if (b + j) % 2 else c.pages + 7
    c.bt = c.table(tables)
    c.ctx = torch.tensor(keys, dtype=torch.int32)
    c.qs = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    c.q = torch.randn(sum(rows), hq, d, generator=c.gen).to(dtype)
    return c.finish(iva, dev)


def cross(iva, dev, c, **kw):
    return iva.paged_cross_attention(c.q.to(dev), *c.pools, c.bt.to(dev), c.ctx.to(dev), c.qs.to(dev), **c.kw, **kw)


def cross_ref(c, scale=None):
    return orc.cross_attention(to_np(c.q), *c.np_pools, c.bt.numpy(), c.ctx.numpy(), c.qs.numpy(), scale=scale)


TYPES = [(t, False) for t in DTYPES] + [(torch.float16, True), (torch.bfloat16, True)]
IDS = ["fp16", "bf16", "fp32", "fp16-fp8", "bf16-fp8"]


@pytest.mark.parametrize("dtype,fp8", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [
    ([1, 1, 1, 1], [1, 16, 37, 300]),            # single-token step
    ([5, 0, 3, 9], [77, 50, 0, 129]),            # a sequence without rows, one without keys
    ([40, 1, 17], [450, 33, 700]),               # several row chunks, segments that are joined
], ids=["steps", "ragged", "long"])
def test_cross_vs_oracle(iva, dev, dtype, fp8, d, rows, keys):
    c = cross_case(iva, dev, rows, keys, 8, 2, d, dtype, fp8, seed=d + len(rows))
    c.check(cross(iva, dev, c), cross_ref(c), f"{dtype} fp8={fp8} D={d}")


@pytest.mark.parametrize("heads", [(4, 4), (12, 4), (16, 1), (40, 2)], ids=str)
def test_cross_heads(iva, dev, heads):
    """Groups of 1, 3, 16 and 20 query heads per kv head."""
    c = cross_case(iva, dev, [3, 7, 1], [90, 260, 5], *heads, 64, torch.bfloat16, seed=3)
    c.check(cross(iva, dev, c), cross_ref(c), str(heads))


@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.3])
def test_cross_scales(iva, dev, scale):
    c = cross_case(iva, dev, [3, 7], [90, 260], 8, 2, 64, torch.float16, seed=4)
    c.check(cross(iva, dev, c, scale=scale), cross_ref(c, scale), f"scale {scale}")


def test_cross_invalid_pages(iva, dev):
    """Keys on an id outside the pool are not attended; a row whose every page is invalid is zero."""
    c = cross_case(iva, dev, [4, 4, 2], [100, 300, 16], 8, 2, 128, torch.float16, seed=5,
                   holes=[(0, 2), (1, 0), (1, 18), (1, 9), (2, 0)])
    out = cross(iva, dev, c)
    c.check(out, cross_ref(c), "holes")
    assert not out[8:].any()


def test_cross_rows_of_no_sequence_stay(iva, dev):
    """Rows outside query_start's range, and rows past max_query_len, keep what out held; a
    strided q is taken as it is."""
    c = cross_case(iva, dev, [4, 3], [60, 200], 8, 2, 64, torch.float16, seed=6)
    q = torch.zeros(11, 8, 128, dtype=torch.float16)
    q[2:9, :, ::2] = c.q
    qs = torch.tensor([2, 6, 9], dtype=torch.int32)
    out = torch.full((11, 8, 64), 7.0, dtype=torch.float16, device=dev)
    iva.paged_cross_attention(q.to(dev)[:, :, ::2], *c.pools, c.bt.to(dev), c.ctx.to(dev), qs.to(dev),
                              max_query_len=4, out=out)
    assert (out[:2] == 7).all() and (out[9:] == 7).all()
    c.check(out[2:9], cross_ref(c), "rows in the middle")


def test_cross_many_sequences(iva, dev):
    """More sequences than a wave has lanes, most of them empty or of one key."""
    keys = [(i * 7) % 50 if i % 3 else i % 2 for i in range(150)]
    rows = [(i * 5) % 4 for i in range(150)]
    c = cross_case(iva, dev, rows, keys, 4, 2, 64, torch.bfloat16, seed=7)
    c.check(cross(iva, dev, c), cross_ref(c), "150 sequences")


# ------------------------------------------------------------------ shared prefixes

def prefix_case(iva, dev, groups, hq, hkv, d, dtype, fp8=False, seed=0, loose=(), width=None):
    """groups: (prefix tokens, [own tokens of each row]); negative own tokens make a row shorter than the
    prefix.  loose: lengths of rows of no group, after the groups."""
    pages = sum(-(-p // 16) + sum(-(-max(p + o, 0) // 16) for o in owns) for p, owns in groups)
    c = Case(iva, pages + sum(-(-n // 16) for n in loose), hkv, d, dtype, fp8, seed)
    rows, lengths, starts, prefixes = [], [], [0], []
    for p, owns in groups:
        shared = c.take(p // 16 * 16)
        for o in owns:
            n = max(p + o, 0)
            rows.append((shared + c.take(max(n - p // 16 * 16, 0)))[:-(-n // 16)])
            lengths.append(n)
        starts.append(len(rows))
        prefixes.append(p)
    for n in loose:
        rows.append(c.take(n))
        lengths.append(n)
    # (a row shorter than the prefix has only its own pages in its table)
    c.bt = c.table(rows, width)
    c.ctx = torch.tensor(lengths, dtype=torch.int32)
    c.gs = torch.tensor(starts, dtype=torch.int32)
    c.pl = torch.tensor(prefixes, dtype=torch.int32)
    c.q = torch.randn(len(rows), hq, d, generator=c.gen).to(dtype)
    return c.finish(iva, dev)


def prefix(iva, dev, c, **kw):
    return iva.paged_prefix_decode_attention(c.q.to(dev), *c.pools, c.bt.to(dev), c.ctx.to(dev), c.gs.to(dev),
                                             c.pl.to(dev), **c.kw, **kw)


def prefix_ref(c, **kw):
    return orc.decode_attention(to_np(c.q), *c.np_pools, c.bt.numpy(), c.ctx.numpy(), **kw)


GROUPS = {
    "one": [(200, [1, 40, 0, 77])],
    "ragged": [(333, [5, 0, 61]), (16, [300]), (700, list(range(0, 90, 9))), (15, [1, 1, 20])],
    "short-rows": [(128, [10, -30, -128, 3])],
}


@pytest.mark.parametrize("dtype,fp8", TYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("name", list(GROUPS))
def test_prefix_vs_oracle(iva, dev, dtype, fp8, d, name):
    c = prefix_case(iva, dev, GROUPS[name], 8, 2, d, dtype, fp8, seed=d)
    c.check(prefix(iva, dev, c), prefix_ref(c), f"{name} {dtype} fp8={fp8} D={d}")


@pytest.mark.parametrize("heads", [(4, 4), (12, 4), (8, 1), (40, 2)], ids=str)
def test_prefix_heads(iva, dev, heads):
    c = prefix_case(iva, dev, GROUPS["ragged"], *heads, 64, torch.float16, seed=8, loose=[45, 0])
    c.check(prefix(iva, dev, c), prefix_ref(c), str(heads))


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (100, 4), (100, 40), (400, 17), (5000, 3), (64, 1000)])
@pytest.mark.parametrize("dtype,fp8", [(torch.float16, False), (torch.bfloat16, True)], ids=["fp16", "bf16-fp8"])
def test_prefix_windows(iva, dev, window, sinks, dtype, fp8):
    """Windows that end inside the prefix, inside the rows' own tokens, and before both; sinks that
    end inside a page."""
    groups = [(500, [1, 300, 37, 0]), (96, [20, 500]), (333, [-100, 40])]
    c = prefix_case(iva, dev, groups, 8, 2, 64, dtype, fp8, seed=window, loose=[250])
    c.check(prefix(iva, dev, c, window=window, n_sink=sinks), prefix_ref(c, window=window, n_sink=sinks),
            f"window {window} sinks {sinks}")


def test_prefix_nan_outside_the_window(iva, dev):
    """A key outside one row's window but inside another's may be NaN: only the rows that see it
    are NaN."""
    c = prefix_case(iva, dev, [(160, [0, 60])], 4, 2, 64, torch.float16, seed=9)
    page, slot = int(c.bt[0, 5]), 3  # position 83: row 0 sees it under a window of 100, row 1 does not
    for i, t in enumerate(c.pools):
        (t[page, :, :, slot] if i == 0 else t[page, :, :, slot])[...] = float("nan")
    out = prefix(iva, dev, c, window=100)
    assert torch.isnan(out[0]).all()
    ref = prefix_ref(c, window=100)
    assert np.isfinite(to_np(out[1])).all()
    assert np.abs(to_np(out[1]) - ref[1]).max() <= 2 * 2.0 ** -11 * 6


def test_prefix_invalid_pages(iva, dev):
    """Invalid ids among the shared pages (in the first row's table and the others'), and among own
    pages; a whole prefix of them."""
    c = prefix_case(iva, dev, [(160, [20, 40]), (64, [0, 30])], 8, 2, 128, torch.bfloat16, seed=10)
    c.bt[0:2, 3] = -1
    c.bt[0:2, 8] = c.pages + 1
    c.bt[1, 11] = -5
    c.bt[2:4, :4] = -1
    c.check(prefix(iva, dev, c), prefix_ref(c), "holes")
    assert not prefix(iva, dev, c)[2].any()


def test_prefix_against_decode(iva, dev):
    """No group at all, groups of one row, and groups that are passed a smaller max_group than they
    have: the same attention as paged_decode_attention."""
    c = prefix_case(iva, dev, [(200, [3, 100, 7, 8, 9])], 8, 2, 128, torch.float16, seed=11)
    ref = prefix_ref(c)
    c.check(prefix(iva, dev, c, max_group=2), ref, "max_group 2")
    c.check(prefix(iva, dev, c, max_group=0), ref, "max_group 0")
    c.check(prefix(iva, dev, c, max_group=1 << 20), ref, "max_group past the batch")
    c.gs, c.pl = torch.arange(6, dtype=torch.int32), torch.full((5,), 200, dtype=torch.int32)
    c.check(prefix(iva, dev, c), ref, "groups of one")
    c.gs, c.pl = torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    c.check(prefix(iva, dev, c), ref, "no groups")
    c.gs, c.pl = torch.tensor([1, 3], dtype=torch.int32), torch.tensor([1 << 30], dtype=torch.int32)
    c.ctx[1:3] = 100  # shorter than the table's pages: nothing is shared
    c.check(prefix(iva, dev, c), prefix_ref(c), "prefix past the table")


def test_prefix_many_groups(iva, dev):
    groups = [((i * 13) % 70, [(i * k) % 40 for k in range(1, 1 + i % 4)]) for i in range(140)]
    c = prefix_case(iva, dev, groups, 4, 2, 64, torch.bfloat16, seed=12)
    c.check(prefix(iva, dev, c), prefix_ref(c), "140 groups")


def test_row_ops_graph_and_streams(iva, dev):
    """Captured and replayed with other lengths and queries; two graphs captured on one stream and
    replayed on two; a side stream with its own workspace: always the eager bits."""
    c = prefix_case(iva, dev, GROUPS["ragged"], 8, 2, 128, torch.float16, seed=13)
    x = cross_case(iva, dev, [40, 3], [450, 129], 8, 2, 128, torch.float16, seed=14)
    q, ctx, xq = c.q.to(dev), c.ctx.to(dev), x.q.to(dev)
    bt, gs, pl = c.bt.to(dev), c.gs.to(dev), c.pl.to(dev)
    xt = [t.to(dev) for t in (x.bt, x.ctx, x.qs)]

    def both():
        return (iva.paged_prefix_decode_attention(q, *c.pools, bt, ctx, gs, pl, max_group=10),
                iva.paged_cross_attention(xq, *x.pools, *xt, max_query_len=40))

    both()
    stream = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(stream):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs = both()
            graphs.append((g, outs))
    torch.cuda.synchronize()
    others = [stream, torch.cuda.Stream()]
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=c.gen).half())
        xq.mul_(0.9)
        ctx.sub_((ctx > 350).int())
        want = [t.clone() for t in both()]
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), step
        with torch.cuda.stream(others[1]):
            side = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(side, want)), step


def test_row_ops_need_sizes_under_capture(iva, dev):
    c = prefix_case(iva, dev, GROUPS["one"], 8, 2, 64, torch.float16, seed=15)
    args = [t.to(dev) for t in (c.bt, c.ctx, c.gs, c.pl)]
    q = c.q.to(dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q.add_(0)
        with pytest.raises(ValueError, match="max_group is required"):
            iva.paged_prefix_decode_attention(q, *c.pools, *args)
        with pytest.raises(ValueError, match="max_query_len is required"):
            iva.paged_cross_attention(q, *c.pools, args[0], args[1], torch.arange(5, dtype=torch.int32, device=dev))


def test_row_ops_device_refusals(iva, dev):
    """Refusals that need the device: rises that are read back, workspaces too small or elsewhere."""
    c = prefix_case(iva, dev, GROUPS["one"], 8, 2, 64, torch.float16, seed=16)
    c.gs = torch.tensor([0, 9], dtype=torch.int32)
    with pytest.raises(ValueError, match="group_start must rise"):
        prefix(iva, dev, c)
    c.gs = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="needed"):
        prefix(iva, dev, c, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    x = cross_case(iva, dev, [2, 2], [20, 30], 8, 2, 64, torch.float16, seed=17)
    x.qs = torch.tensor([0, 3, 2], dtype=torch.int32)
    with pytest.raises(ValueError, match="query_start must rise"):
        cross(iva, dev, x)
    x.qs = torch.tensor([0, 2, 4], dtype=torch.int32)
    n = iva.cross_workspace_bytes(2, 4, 2, 8, 2, 64, x.bt.shape[1], torch.float16)
    ws = torch.full((n + 256,), 0x7F, dtype=torch.uint8, device=dev)
    x.check(cross(iva, dev, x, workspace=ws[:n], max_query_len=2), cross_ref(x), "own workspace")
    assert (ws[n:] == 0x7F).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d,rows,keys", [(128, [70, 65, 130], [333, 0, 200]), (256, [40, 1, 33], [130, 300, 17])])
def test_cross_many_rows(iva, dev, dtype, d, rows, keys):
    """Enough whole row chunks to be walked through LDS (32 kv heads), with an invalid page, a sequence
    without keys and rows past the last whole chunk."""
    c = cross_case(iva, dev, rows + [64] * 8, keys + [40] * 8, 128, 32, d, dtype, seed=20, holes=[(0, 3)])
    c.check(cross(iva, dev, c), cross_ref(c), f"{dtype} D={d}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_prefix_many_rows(iva, dev, dtype):
    """A prefix of pieces walked through LDS: 320 rows per kv head on a wide table, rows that take
    part and rows that do not, a ragged second group."""
    groups = [(1000, [i % 23 for i in range(78)] + [-500, -1000]), (333, [3] * 21)]
    c = prefix_case(iva, dev, groups, 4, 1, 128, dtype, seed=21, width=1100)
    c.check(prefix(iva, dev, c), prefix_ref(c), str(dtype))
    c.check(prefix(iva, dev, c, window=1005, n_sink=3), prefix_ref(c, window=1005, n_sink=3), "window")
