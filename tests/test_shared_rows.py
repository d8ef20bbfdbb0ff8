"""Refusals of the cross-attention, shared-prefix and log-probability entry points and ops, without a
GPU: every call fails before a kernel would start, or has nothing to do."""
from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 0x10000  # a 16-byte-aligned non-null address; never dereferenced by these calls


def call(iva, name, *args):
    return getattr(iva._abi.lib(), name)(*args)


def cross_args(iva, **over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, bt=FAKE, ctx=FAKE, qs=FAKE, n_tok=8, out=FAKE, ws=FAKE,
                ws_bytes=1 << 40, batch=2, hq=8, hkv=2, d=128, bs=16, max_blocks=8, num_pages=16, max_q=4,
                scale=0.1, dtype=iva._abi.F16, stream=None)
    args.update(over)
    return list(args.values())


def prefix_args(iva, **over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, ks=None, vs=None, bt=FAKE, ctx=FAKE, gs=FAKE, pl=FAKE, groups=1, out=FAKE,
                ws=FAKE, ws_bytes=1 << 40, batch=2, hq=8, hkv=2, d=128, bs=16, max_blocks=8, num_pages=16,
                max_group=2, scale=0.1, window=0, n_sink=0, dtype=iva._abi.F16, stream=None)
    args.update(over)
    return list(args.values())


@pytest.mark.parametrize("name,build", [("ivakv_cross_attn", cross_args), ("ivakv_prefix_decode_attn", prefix_args)])
def test_row_entry_refusals(iva, name, build):
    a = iva._abi
    for over, status in [
            (dict(dtype=3), a.E_DTYPE), (dict(dtype=a.F32, ks=FAKE, vs=FAKE), a.E_DTYPE),
            (dict(bs=32), a.E_SHAPE), (dict(d=96), a.E_SHAPE), (dict(hq=9), a.E_SHAPE),
            (dict(hkv=0), a.E_ARG), (dict(batch=-1), a.E_ARG), (dict(max_blocks=-1), a.E_ARG),
            (dict(num_pages=0), a.E_ARG), (dict(q=None), a.E_ARG), (dict(out=None), a.E_ARG),
            (dict(bt=None), a.E_ARG), (dict(ctx=None), a.E_ARG), (dict(k=FAKE + 8), a.E_ARG),
            (dict(ks=FAKE), a.E_ARG), (dict(ks=FAKE, vs=FAKE + 4), a.E_ARG), (dict(scale=float("nan")), a.E_ARG),
            (dict(ws=None), a.E_WORKSPACE), (dict(ws_bytes=64), a.E_WORKSPACE), (dict(ws=FAKE + 4), a.E_WORKSPACE),
            (dict(hq=1 << 30, hkv=1 << 30, n_tok=1 << 20) if name == "ivakv_cross_attn" else
             dict(hq=1 << 30, hkv=1 << 30, batch=1 << 20), a.E_SHAPE),
            *([] if name == "ivakv_cross_attn" else [(dict(batch=8193), a.E_SHAPE), (dict(max_blocks=1 << 30), a.E_SHAPE)])]:
        assert call(iva, name, *build(iva, **over)) == status, over
        assert name in a.last_error()


def test_row_entries_with_nothing_to_do(iva):
    a = iva._abi
    nothing = dict(q=None, k=None, v=None, out=None, ctx=None, bt=None)
    assert call(iva, "ivakv_cross_attn", *cross_args(iva, batch=0, **nothing)) == a.OK
    assert call(iva, "ivakv_cross_attn", *cross_args(iva, n_tok=0, **nothing)) == a.OK
    assert call(iva, "ivakv_cross_attn", *cross_args(iva, max_q=0, **nothing)) == a.OK
    assert call(iva, "ivakv_prefix_decode_attn", *prefix_args(iva, batch=0, **nothing)) == a.OK
    assert call(iva, "ivakv_prefix_decode_attn", *prefix_args(iva, n_sink=-1)) == a.E_ARG
    assert call(iva, "ivakv_prefix_decode_attn", *prefix_args(iva, pl=None)) == a.E_ARG
    assert call(iva, "ivakv_prefix_decode_attn", *prefix_args(iva, gs=None)) == a.E_ARG


def test_row_workspace_sizes(iva):
    a = iva._abi
    n = ctypes.c_size_t(7)
    for name in ("ivakv_cross_workspace_size", "ivakv_prefix_workspace_size"):
        assert call(iva, name, 2, 8, 4, 8, 2, 100, 9, a.F16, 0, ctypes.byref(n)) == a.E_SHAPE and n.value == 0
        assert call(iva, name, 2, 8, 4, 8, 2, 128, 9, 9, 0, ctypes.byref(n)) == a.E_DTYPE
        assert call(iva, name, 2, 8, 4, 8, 2, 128, 9, a.F16, 0, None) == a.E_ARG
        assert call(iva, name, 2, 8, 4, 8, 3, 128, 9, a.F16, 0, ctypes.byref(n)) == a.E_SHAPE
    assert call(iva, "ivakv_prefix_workspace_size", 2, 1, 2, 8, 2, 128, -1, a.F16, 0, ctypes.byref(n)) == a.E_ARG
    # grows with nothing but the launch: no rows, no partials
    assert iva.cross_workspace_bytes(0, 0, 0, 8, 2, 128, 100, torch.float16) == 0
    assert iva.prefix_workspace_bytes(0, 0, 0, 8, 2, 128, 100, torch.float16) == 0
    wide, narrow = (iva.prefix_workspace_bytes(64, 1, 64, 32, 8, 128, n, torch.float16) for n in (1000, 1))
    assert wide > narrow > 0


def pools(iva, dtype=torch.float16):
    return [torch.zeros(s, dtype=dtype) for s in iva.pool_shapes(4, 2, 64, 16, dtype)]


def test_row_ops_refuse_cpu_tensors(iva):
    q, i = torch.zeros(2, 4, 64, dtype=torch.float16), lambda *x: torch.tensor(x, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        iva.paged_cross_attention(q, *pools(iva), i(0, 1).view(2, 1), i(3, 3), i(0, 1, 2))
    with pytest.raises(RuntimeError, match="GPU"):
        iva.paged_prefix_decode_attention(q, *pools(iva), i(0, 1).view(2, 1), i(3, 3), i(0, 2), i(16))
    with pytest.raises(RuntimeError, match="GPU"):
        iva.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


def logprob_args(iva, **over):
    args = dict(logits=FAKE, stride=100, tokens=FAKE, n=3, vocab=100, top=5, lp=FAKE, h=FAKE, stats=None, tl=FAKE,
                tt=FAKE, dtype=iva._abi.BF16, stream=None)
    args.update(over)
    return list(args.values())


def grad_args(iva, **over):
    args = dict(logits=FAKE, stride=100, tokens=FAKE, h=FAKE, stats=FAKE, tt=FAKE, g=FAKE, gh=FAKE, gt=FAKE, n=3,
                vocab=100, top=5, grad=FAKE, dtype=iva._abi.BF16, stream=None)
    args.update(over)
    return list(args.values())


@pytest.mark.parametrize("name,build", [("ivakv_token_logprobs", logprob_args),
                                        ("ivakv_token_logprobs_grad", grad_args)])
def test_logprob_entry_refusals(iva, name, build):
    a = iva._abi
    for over, status in [
            (dict(dtype=7), a.E_DTYPE), (dict(n=-1), a.E_ARG), (dict(vocab=-1), a.E_ARG), (dict(stride=-1), a.E_ARG),
            (dict(top=-1), a.E_ARG), (dict(top=65), a.E_SHAPE), (dict(top=6, vocab=5), a.E_SHAPE),
            (dict(vocab=0, top=0), a.E_SHAPE), (dict(n=1 << 40), a.E_SHAPE), (dict(logits=None), a.E_ARG),
            (dict(logits=FAKE + 1), a.E_ARG), (dict(tokens=None), a.E_ARG), (dict(tt=None), a.E_ARG),
            (dict(h=None), a.E_ARG)]:
        assert call(iva, name, *build(iva, **over)) == status, over
        assert name in a.last_error()
    assert call(iva, name, *build(iva, n=0, logits=None, tokens=None, h=None)) == a.OK


def test_launches_past_the_grid_are_refused(iva):
    """A grid has less than 2^32 threads."""
    a = iva._abi
    for name, build in (("ivakv_token_logprobs", logprob_args), ("ivakv_token_logprobs_grad", grad_args)):
        assert call(iva, name, *build(iva, n=1 << 24)) == a.E_SHAPE and str((1 << 24) - 1) in a.last_error()
    # (cut into pieces: a join of every row and kv head)
    assert call(iva, "ivakv_cross_attn", *cross_args(iva, n_tok=1 << 22, hq=4, hkv=4, max_q=1)) == a.E_SHAPE
    assert call(iva, "ivakv_cross_attn", *cross_args(iva, n_tok=1 << 28, hq=4, hkv=4, max_q=1 << 28)) == a.E_SHAPE


class _Device:
    """Stands for a GPU tensor in the ops' argument checks."""
    is_cuda, device, requires_grad = True, torch.device("cuda", 0), False

    def __init__(self, *shape, dtype=torch.float16):
        self.shape, self.dtype = torch.Size(shape), dtype

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return True

    def contiguous(self):
        return self


@pytest.mark.parametrize("what,kw,error", [
    ("tokens' shape", dict(tokens=(3,)), ValueError), ("tokens' type", dict(t_dtype=torch.float32), TypeError),
    ("logits' type", dict(dtype=torch.float64), TypeError), ("tops past the vocabulary", dict(k=9), ValueError),
    ("tops past 64", dict(k=65, v=100), ValueError), ("negative tops", dict(k=-1), ValueError)])
def test_logprob_op_refusals(iva, what, kw, error):
    logits = _Device(2, kw.get("v", 8), dtype=kw.get("dtype", torch.float16))
    tokens = _Device(*kw.get("tokens", (2,)), dtype=kw.get("t_dtype", torch.int64))
    with pytest.raises(error):
        iva.token_logprobs(logits, tokens, kw.get("k", 0))


@pytest.mark.parametrize("what,change,error", [
    ("q's dims", dict(q=(2, 4, 32)), ValueError), ("q's type", dict(q_dtype=torch.bfloat16), TypeError),
    ("a table of other rows", dict(bt=(3, 1)), ValueError), ("starts of other groups", dict(start=(5,)), ValueError),
    ("a table of another type", dict(bt_dtype=torch.int64), TypeError), ("an out of another shape", dict(out=(2, 4, 65)), ValueError)])
@pytest.mark.parametrize("op", ["cross", "prefix"])
def test_row_op_refusals(iva, op, what, change, error):
    i32 = dict(dtype=torch.int32)
    q = _Device(*change.get("q", (2, 4, 64)), dtype=change.get("q_dtype", torch.float16))
    kp, vp = _Device(4, 2, 8, 16, 8), _Device(4, 2, 64, 16)
    bt = _Device(*change.get("bt", (2, 1)), dtype=change.get("bt_dtype", torch.int32))
    start = _Device(*change.get("start", (3,) if op == "cross" else (2,)), **i32)
    out = _Device(*change["out"]) if "out" in change else _Device(2, 4, 64)
    with pytest.raises(error):
        if op == "cross":
            iva.paged_cross_attention(q, kp, vp, bt, _Device(2, **i32), start, max_query_len=1, out=out)
        else:
            iva.paged_prefix_decode_attention(q, kp, vp, bt, _Device(2, **i32), start, _Device(1, **i32), max_group=2,
                                              out=out)


def test_capture_beside_a_live_eager_graph_is_refused(iva, monkeypatch):
    """The check alone, on a leaf of the host with stand-ins for the stream and its state."""
    ops, now = iva.ops, {"stream": 0, "capturing": False}
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now["stream"])
    monkeypatch.setattr(ops, "_capturing", lambda dev: now["capturing"])
    dev, leaf = torch.device("cuda", 0), torch.randn(2, 3, requires_grad=True)

    def call():
        node = ops._same_stream_as_before(leaf, dev)
        out = leaf.sum()  # (holds the leaf's gradient node)
        del node
        return out

    eager = call()
    now.update(stream=7)
    assert call() is not None  # another stream, but no capture
    now.update(capturing=True)
    with pytest.raises(RuntimeError, match="eager graph"):
        call()
    now.update(stream=0)
    assert call() is not None  # the same stream
    del eager
    now.update(stream=7)
    assert call() is not None  # the eager graph is gone
