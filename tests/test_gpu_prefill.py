"""GPU checks of paged_prefill and varlen_attention against 64 bits: types, head
layouts, rows from none to many tokens, masks, strides, and what lies where no
token looks."""

from __future__ import annotations

import math

import pytest
import torch

from tests import prefill_oracle as po
from vllm_fastdecoder_amd import ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
# (query heads, kv heads, head size)
LAYOUTS = [(4, 4, 128), (8, 2, 128), (7, 1, 64), (6, 2, 80), (4, 2, 96), (4, 2, 256), (3, 1, 112),
           (4, 1, 48), (8, 8, 32), (2, 1, 72), (2, 2, 20), (2, 1, 192)]
# rows of (new tokens, tokens in all)
RAGGED = [(1, 1), (1, 77), (5, 5), (0, 40), (17, 17), (33, 300), (130, 131), (64, 64), (2, 513)]


def _run_paged(p, scale, causal=True, out_dtype=None, max_k=None, dev="cuda", **kw):
    kv = p.kv.to(dev)
    out = lse = None
    if out_dtype is not None:
        out = torch.full((p.T,) + tuple(p.q.shape[1:]), 7.0, dtype=out_dtype, device=dev)
        lse = torch.full((p.q.shape[1], p.T), 7.0, device=dev)
    return ops.paged_prefill(p.q.to(dev), kv[..., :p.D], kv[..., p.D:], p.bt.to(dev), p.cu.to(dev),
                             p.lens.to(dev), scale, max_seqlen_q=max(p.qs, default=0),
                             max_seqlen_k=max_k if max_k is not None else max(p.ks, default=0),
                             causal=causal, out=out, lse=lse, **kw)


def _check_paged(p, out, lse, scale, causal, what=""):
    for q0, nq, ref in p.refs(scale, causal, out.dtype):
        po.check(out[q0:q0 + nq], lse[:, q0:q0 + nq], ref, f"{what} row at {q0}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_paged_rows_of_every_length(gpu, layout, dtype):
    H, KVH, D = layout
    p = po.Paged([q for q, _ in RAGGED], [k for _, k in RAGGED], H, KVH, D, dtype, seed=D + H,
                 extra_cols=3)
    scale = 1 / math.sqrt(D)
    out, lse = _run_paged(p, scale)
    _check_paged(p, out, lse, scale, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("qs,ks", [
    ([300], [300]), ([257], [1000]), ([1], [4000]), ([3] * 9, [50, 64, 65, 1, 2, 3, 700, 31, 33]),
    ([1] * 20, list(range(1, 400, 20))), ([40, 1, 1, 200, 1], [40, 600, 3, 333, 129])], ids=str)
def test_paged_lengths(gpu, dtype, causal, qs, ks):
    if not causal:
        ks = [k + 5 for k in ks]
    p = po.Paged(qs, ks, 8, 2, 64, dtype, seed=1)
    out, lse = _run_paged(p, 0.125, causal=causal, out_dtype=torch.float32)
    _check_paged(p, out, lse, 0.125, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("BS", [1, 8, 16, 24, 32, 64, 256])
def test_block_sizes(gpu, dtype, BS):
    """Blocks smaller and larger than the kernels' steps, and not powers of two."""
    p = po.Paged([5, 150, 1], [100, 420, 300], 4, 2, 64, dtype, BS=BS, seed=BS)
    out, lse = _run_paged(p, 0.125)
    _check_paged(p, out, lse, 0.125, True, f"BS {BS}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_keys(gpu, dtype):
    """More new tokens than tokens in all: the first ones see nothing."""
    p = po.Paged([40, 3, 200, 2], [10, 0, 64, 1], 4, 2, 128, dtype, seed=3)
    out, lse = _run_paged(p, 0.1)
    _check_paged(p, out, lse, 0.1, True)
    assert torch.all(out[:30] == 0) and torch.all(torch.isneginf(lse[:, :30]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_are_left_alone(gpu, dtype):
    p = po.Paged([20, 9], [100, 9], 8, 2, 64, dtype, seed=4, pad=13)
    out, lse = _run_paged(p, 0.125, out_dtype=torch.float32)
    _check_paged(p, out, lse, 0.125, True)
    assert torch.all(out[29:] == 7.0) and torch.all(lse[:, 29:] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-8, 3.0])
def test_scales(gpu, dtype, scale):
    p = po.Paged([70, 4], [200, 90], 4, 2, 64, dtype, seed=5)
    out, lse = _run_paged(p, scale, out_dtype=torch.float32)
    _check_paged(p, out, lse, scale, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qs,ks", [([150], [150]), ([3], [40]), ([90], [300])], ids=str)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_only_who_sees_them(gpu, dtype, qs, ks, bad):
    """A key and a value of a late token: earlier tokens of the row do not see them."""
    p = po.Paged(qs, ks, 4, 2, 64, dtype, seed=6)
    nk = ks[0]
    at = nk - min(qs[0], 40) // 2 - 1
    blk, off = int(p.bt[0, at // p.BS]), at % p.BS
    p.v[0][at, 0, 3] = bad
    p.v[0][at, 1, 60] = bad
    p.kv[blk, off, :, 64:] = p.v[0][at]
    out, lse = _run_paged(p, 0.125)
    _check_paged(p, out, lse, 0.125, True, f"V {bad}")
    p.v[0][at] = 1.0
    p.k[0][at] = math.nan  # (a NaN key: every score with it is NaN)
    p.kv[blk, off, :, :64] = p.k[0][at]
    p.kv[blk, off, :, 64:] = p.v[0][at]
    out, lse = _run_paged(p, 0.125)
    first = qs[0] - (nk - at)  # the first token that sees it
    ref = po.attend(p.q[:first], p.k[0][:at], p.v[0][:at], 0.125, True, out.dtype)
    po.check(out[:first], lse[:, :first], ref, "K NaN")
    assert torch.isnan(out[first:]).all() and torch.isnan(lse[:, first:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(gpu, dtype):
    """Scores of some hundreds, whose weights are mostly nothing, and a growing maximum."""
    p = po.Paged([100, 2], [400, 700], 4, 2, 128, dtype, seed=7, amp=12.0)
    out, lse = _run_paged(p, 0.3, out_dtype=torch.float32)
    _check_paged(p, out, lse, 0.3, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("layout", [(4, 4, 64), (8, 2, 128), (2, 1, 40), (20, 4, 80), (4, 2, 256)],
                         ids=str)
def test_packed_rows(gpu, dtype, causal, layout):
    """Fresh prompts and cross attention over strided views of fused projections."""
    H, KVH, D = layout
    g = torch.Generator().manual_seed(11)
    qs, ks = [1, 60, 0, 7, 140, 33], [90, 60, 10, 0, 150, 500]
    if causal:
        ks = qs
    T, Tk = sum(qs), sum(ks)
    q = torch.randn(T, 2, H, D, generator=g).to(dtype)[:, 1]
    kv = torch.randn(Tk, KVH, 2, D, generator=g).to(dtype)
    scale = 1 / math.sqrt(D)
    out, lse = ops.varlen_attention(q.to(gpu), kv.to(gpu)[:, :, 0], kv.to(gpu)[:, :, 1],
                                    po.starts(qs).to(gpu), po.starts(ks).to(gpu), scale,
                                    max_seqlen_q=max(qs), max_seqlen_k=max(ks), causal=causal)
    q0 = k0 = 0
    for nq, nk in zip(qs, ks):
        ref = po.attend(q[q0:q0 + nq], kv[k0:k0 + nk, :, 0], kv[k0:k0 + nk, :, 1], scale, causal,
                        out.dtype)
        po.check(out[q0:q0 + nq], lse[:, q0:q0 + nq], ref, f"row at {q0}")
        q0 += nq
        k0 += nk


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(gpu, dtype):
    """Heads ahead of tokens, rows that no 16-byte load may start at, an output inside a larger one."""
    H, KVH, D = 4, 2, 64
    p = po.Paged([50, 3], [90, 200], H, KVH, D, dtype, seed=12)
    kv = p.kv.to(gpu)
    wide = torch.empty(p.B, p.BS, KVH, 2 * D + 1, dtype=dtype, device=gpu)
    wide[..., :2 * D] = kv
    q = torch.empty(H, p.T, D + 1, dtype=dtype, device=gpu)
    q[..., :D] = p.q.to(gpu).transpose(0, 1)
    big = torch.zeros(p.T + 2, H, D + 3, dtype=dtype, device=gpu)
    host_tier = kv.transpose(1, 2).contiguous()  # [B, KVH, BS, 2D]
    for qq, k, v, out in (
            (p.q.to(gpu), wide[..., :D], wide[..., D:2 * D], None),
            (q.transpose(0, 1)[..., :D], kv[..., :D], kv[..., D:], None),
            (p.q.to(gpu), kv[..., :D], kv[..., D:], big[1:-1, :, 1:-2]),
            (p.q.to(gpu), host_tier.transpose(1, 2)[..., :D], host_tier.transpose(1, 2)[..., D:], None)):
        o, lse = ops.paged_prefill(qq, k, v, p.bt.to(gpu), p.cu.to(gpu), p.lens.to(gpu), 0.125,
                                   max_seqlen_q=50, max_seqlen_k=200, out=out)
        _check_paged(p, o, lse, 0.125, True)
    assert torch.all(big[0] == 0) and torch.all(big[-1] == 0) and torch.all(big[..., 0] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [2, 100])
def test_range_errors_make_the_row_nan(gpu, dtype, nq):
    """A block id outside the cache, a length past the table, more tokens than max_seqlen_q: that
    row is NaN, the others are right."""
    p = po.Paged([nq, nq, nq, nq], [120, 200, 150, 180], 4, 2, 64, dtype, seed=13)
    bt = p.bt.clone()
    bt[1, 12] = p.B  # read by the row's last tokens only
    kv = p.kv.to(gpu)
    lens = p.lens.clone()
    lens[3] = 13 * 16 + 1
    out, lse = ops.paged_prefill(p.q.to(gpu), kv[..., :64], kv[..., 64:], bt.to(gpu),
                                 p.cu.to(gpu), lens.to(gpu), 0.125, max_seqlen_q=nq,
                                 max_seqlen_k=13 * 16)
    for i, (q0, m, ref) in enumerate(p.refs(0.125, True, out.dtype)):
        if i in (1, 3):
            assert torch.isnan(out[q0:q0 + m]).all() and torch.isnan(lse[:, q0:q0 + m]).all()
        else:
            po.check(out[q0:q0 + m], lse[:, q0:q0 + m], ref)
    p = po.Paged([3, nq + 3, nq], [120, 200, 150], 4, 2, 64, dtype, seed=14)
    kv = p.kv.to(gpu)
    out, lse = ops.paged_prefill(p.q.to(gpu), kv[..., :64], kv[..., 64:], p.bt.to(gpu),
                                 p.cu.to(gpu), p.lens.to(gpu), 0.125, max_seqlen_q=max(nq, 3))
    for i, (q0, m, ref) in enumerate(p.refs(0.125, True, out.dtype)):
        if i == 1:
            assert torch.isnan(out[q0:q0 + m]).all() and torch.isnan(lse[:, q0:q0 + m]).all()
        else:
            po.check(out[q0:q0 + m], lse[:, q0:q0 + m], ref)


def test_rows_that_do_not_lie_in_the_tokens_are_not_written(gpu):
    p = po.Paged([20, 9, 30], [100, 9, 30], 8, 2, 64, torch.bfloat16, seed=15)
    cu = p.cu.clone()
    cu[2] = 5  # row 1 ends before it starts, row 2 covers part of row 0's tokens too
    cu[3] = p.T + 40
    kv = p.kv.to(gpu)
    out = torch.full_like(p.q, 7.0).to(gpu)
    lse = torch.full((8, p.T), 7.0, device=gpu)
    ops.paged_prefill(p.q.to(gpu), kv[..., :64], kv[..., 64:], p.bt.to(gpu), cu.to(gpu),
                      p.lens.to(gpu), 0.125, max_seqlen_q=64, out=out, lse=lse)
    ref = next(iter(p.refs(0.125, True, out.dtype)))[2]
    po.check(out[:20], lse[:, :20], ref)
    assert torch.all(out[20:] == 7.0) and torch.all(lse[:, 20:] == 7.0)


def test_empty_calls(gpu):
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=gpu)
    cu = torch.zeros(1, dtype=torch.int32, device=gpu)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device=gpu)
    out, lse = ops.paged_prefill(q, kc, kc, torch.zeros(0, 3, dtype=torch.int32, device=gpu), cu,
                                 cu[:0], 1.0, max_seqlen_q=0)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    # a table without columns, an empty cache, packed keys of no token: rows of no key
    q = torch.ones(3, 4, 64, dtype=torch.float16, device=gpu)
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=gpu)
    none = torch.zeros(2, dtype=torch.int32, device=gpu)
    for cache, cols in ((kc, 0), (kc[:0], 2)):
        out, lse = ops.paged_prefill(q, cache, cache,
                                     torch.zeros(2, cols, dtype=torch.int32, device=gpu), cu, none,
                                     1.0, max_seqlen_q=2)
        assert torch.all(out == 0) and torch.isneginf(lse).all()
    out, lse = ops.varlen_attention(q, q[:0, :2], q[:0, :2], cu, torch.zeros_like(cu), 1.0, 2, 0)
    assert torch.all(out == 0) and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qs,ks", [([4, 1, 9], [3000, 700, 1500]), ([300], [900])], ids=str)
def test_graph_replays_and_other_streams(gpu, dtype, qs, ks):
    """Captured calls (two graphs of one stream, each with its own scratch), replayed with eager
    work in between and other inputs, and a call on a side stream."""
    ps = [po.Paged(qs, ks, 8, 2, 64, dtype, seed=s) for s in (20, 21, 22)]
    dev = [dict(q=p.q.to(gpu), kv=p.kv.to(gpu), bt=p.bt.to(gpu), cu=p.cu.to(gpu), ln=p.lens.to(gpu))
           for p in ps]

    def call(x):
        return ops.paged_prefill(x["q"], x["kv"][..., :64], x["kv"][..., 64:], x["bt"], x["cu"],
                                 x["ln"], 0.125, max_seqlen_q=max(qs), max_seqlen_k=max(ks))

    eager = [call(x) for x in dev]
    for p, (o, l) in zip(ps, eager):
        _check_paged(p, o, l, 0.125, True)
    live = [{k: v.clone() for k, v in dev[0].items()} for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for x in live:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(call(x))
        graphs.append(g)
    for turn in range(4):
        for k, g in enumerate(graphs):
            src = dev[(turn + k) % 3]
            for name, t in live[k].items():
                t.copy_(src[name])
            g.replay()
            call(dev[turn % 3])
        torch.cuda.synchronize()
        for k in range(2):
            want = eager[(turn + k) % 3]
            assert torch.equal(outs[k][0], want[0]) and torch.equal(outs[k][1], want[1])
    with torch.cuda.stream(side):
        o, l = call(dev[1])
    side.synchronize()
    assert torch.equal(o, eager[1][0]) and torch.equal(l, eager[1][1])
