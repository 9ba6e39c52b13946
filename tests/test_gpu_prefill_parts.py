"""GPU checks of the ways a call of paged_prefill / varlen_attention is cut: tiles of eight
waves, keys divided into parts that the last one joins, and the offsets' tables."""

from __future__ import annotations

import math

import pytest
import torch

from tests import prefill_oracle as po
from vllm_fastdecoder_amd import ops
from vllm_fastdecoder_amd.pinned import pinned_zeros

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _run(p, scale=0.125, causal=True, k=None, v=None, bt=None, dev="cuda"):
    kv = p.kv.to(dev)
    return ops.paged_prefill(p.q.to(dev), kv[..., :p.D] if k is None else k,
                             kv[..., p.D:] if v is None else v, (p.bt if bt is None else bt).to(dev),
                             p.cu.to(dev), p.lens.to(dev), scale, max_seqlen_q=max(p.qs),
                             max_seqlen_k=max(p.ks), causal=causal)


def _check(p, out, lse, scale=0.125, causal=True, nan_rows=()):
    for i, (q0, nq, ref) in enumerate(p.refs(scale, causal, out.dtype)):
        if i in nan_rows:
            assert torch.isnan(out[q0:q0 + nq]).all() and torch.isnan(lse[:, q0:q0 + nq]).all()
        else:
            po.check(out[q0:q0 + nq], lse[:, q0:q0 + nq], ref, f"row {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 48, 64, 80, 96, 112, 128])
def test_many_tokens_over_many_keys(gpu, dtype, D):
    """Enough tiles of eight waves for every CU: tokens and heads picked from all over."""
    H, T, L = 34, 2047, 4200
    g = torch.Generator(device="cuda").manual_seed(D)
    q = torch.randn(T, H, D, generator=g, device=gpu).to(dtype)
    k = torch.randn(L, H, D, generator=g, device=gpu).to(dtype)
    v = torch.randn(L, H, D, generator=g, device=gpu).to(dtype)
    cu_q = torch.tensor([0, T], dtype=torch.int32, device=gpu)
    cu_k = torch.tensor([0, L], dtype=torch.int32, device=gpu)
    scale = 1 / math.sqrt(D)
    for causal in (True, False):
        out, lse = ops.varlen_attention(q, k, v, cu_q, cu_k, scale, max_seqlen_q=T, max_seqlen_k=L,
                                        causal=causal)
        for h in (0, 5, 33):
            qc, kc, vc = (x[:, h:h + 1].cpu() for x in (q, k, v))
            for t in (0, 1, 31, 32, 255, 256, 1000, 1791, 1792, 2045, 2046):
                see = L - T + t + 1 if causal else L
                ref = po.attend(qc[t:t + 1], kc[:see], vc[:see], scale, False, out.dtype)
                po.check(out[t:t + 1, h:h + 1], lse[h:h + 1, t:t + 1], ref, f"token {t} head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 80, 128])
def test_rows_of_few_tokens_beside_many(gpu, dtype, D):
    """The same tiles, and short rows' tiles of eight waves beside them."""
    H, qs, ks = 64, [3, 2100, 1, 64], [900, 4200, 1, 4100]
    g = torch.Generator(device="cuda").manual_seed(D)
    q = torch.randn(sum(qs), H, D, generator=g, device=gpu).to(dtype)
    k = torch.randn(sum(ks), H, D, generator=g, device=gpu).to(dtype)
    v = torch.randn(sum(ks), H, D, generator=g, device=gpu).to(dtype)
    cu_q, cu_k = po.starts(qs), po.starts(ks)
    scale = 1 / math.sqrt(D)
    out, lse = ops.varlen_attention(q, k, v, cu_q.to(gpu), cu_k.to(gpu), scale, max_seqlen_q=2100,
                                    max_seqlen_k=4200, causal=True)
    for h in (0, 33, 63):
        qc, kc, vc = (x[:, h:h + 1].cpu() for x in (q, k, v))
        for i, tokens in ((0, (0, 1, 2)), (1, (0, 63, 2047, 2099)), (2, (0,)), (3, (0, 31, 32, 63))):
            for j in tokens:
                t, k0 = int(cu_q[i]) + j, int(cu_k[i])
                see = slice(k0, k0 + ks[i] - qs[i] + j + 1)
                ref = po.attend(qc[t:t + 1], kc[see], vc[see], scale, False, out.dtype)
                po.check(out[t:t + 1, h:h + 1], lse[h:h + 1, t:t + 1], ref, f"row {i} token {j} head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [48, 64, 128, 256])
@pytest.mark.parametrize("qs,ks", [([300], [4100]), ([3], [4100]), ([100, 37, 5], [2900, 40, 1500])],
                         ids=str)
def test_divided_keys(gpu, dtype, D, qs, ks):
    """Few tiles of many keys: every part's sums and their join, the same in every call."""
    p = po.Paged(qs, ks, 6, 2, D, dtype, seed=D)
    out, lse = _run(p)
    _check(p, out, lse)
    again = _run(p)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [4, 120])
@pytest.mark.parametrize("block", [0, 60, 130, 187])
def test_a_bad_block_in_any_part(gpu, dtype, nq, block):
    """Whichever part reads it, and where only the last tokens see it: the whole row is NaN."""
    p = po.Paged([nq, nq], [3000, 2999], 8, 2, 64, dtype, seed=31)
    bt = p.bt.clone()
    bt[1, block] = p.B if block % 20 else -1
    _check(p, *_run(p, bt=bt), nan_rows=(1,))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq", [4, 120])
def test_values_that_are_not_finite_in_a_part(gpu, dtype, nq):
    p = po.Paged([nq, 2], [3000, 70], 4, 2, 64, dtype, seed=32)
    kv = p.kv
    k, v = p.k[0], p.v[0]
    v[1500, 0, 3] = math.inf
    v[2999, 1, 5] = math.nan  # seen by the last token alone
    k[700, 1, :] = 0
    k[700, 1, 0] = math.inf   # a score of +-inf
    for key in (1500, 2999, 700):
        b, at = int(p.bt[0, key // 16]), key % 16
        kv[b, at, :, :64], kv[b, at, :, 64:] = k[key], v[key]
    out, lse = _run(p)
    (q0, n0, ref), (q1, n1, other) = p.refs(0.125, True, out.dtype)
    po.check(out[q1:q1 + n1], lse[:, q1:q1 + n1], other, "the row beside")
    # kv head 0 (heads 0, 1): all but one dim is finite
    half = tuple(x[:, :2] for x in ref)
    po.check(out[:n0, :2], lse[:2, :n0], half, "kv head 0")
    # kv head 1: a query whose first value is negative scores -inf there (weight 0); a positive one
    # +inf, whose weights are not numbers
    first = p.q[:n0, 2:, 0].double()
    got = out[:n0, 2:].cpu()
    assert torch.isnan(got[first > 0]).all()
    quiet = (first < 0)[:-1]
    assert torch.isfinite(got[:-1][quiet]).all()
    assert torch.isnan(got[-1, :, 5]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qs,ks", [([150, 3], [700, 2500]), ([2], [3000]), ([90], [90])], ids=str)
def test_v_laid_out_otherwise_than_k(gpu, dtype, qs, ks):
    H, KVH, D = 4, 2, 64
    g = torch.Generator().manual_seed(33)
    q = torch.randn(sum(qs), H, D, generator=g).to(dtype)
    k = torch.randn(sum(ks), KVH, D, generator=g).to(dtype)
    v = torch.randn(sum(ks), KVH, D, generator=g).to(dtype)
    wide = torch.full((sum(ks), KVH + 1, D + 8), math.nan, dtype=dtype, device=gpu)
    wide[:, :KVH, :D] = v.to(gpu)
    heads_first = k.to(gpu).transpose(0, 1).contiguous().transpose(0, 1)
    cu_q, cu_k = po.starts(qs), po.starts(ks)
    for kk in (k.to(gpu), heads_first):
        out, lse = ops.varlen_attention(q.to(gpu), kk, wide[:, :KVH, :D], cu_q.to(gpu), cu_k.to(gpu),
                                        0.125, max_seqlen_q=max(qs), max_seqlen_k=max(ks), causal=True)
        for i in range(len(qs)):
            a, b, c, d = int(cu_q[i]), int(cu_q[i + 1]), int(cu_k[i]), int(cu_k[i + 1])
            ref = po.attend(q[a:b], k[c:d], v[c:d], 0.125, True, out.dtype)
            po.check(out[a:b], lse[:, a:b], ref, f"row {i}")


def test_more_tasks_than_counters(gpu):
    """Rows by the thousand, one of them longer than a part's table of single-token blocks."""
    n = 2100
    p = po.Paged([1] * n, [3] * (n - 1) + [5000], 2, 1, 64, torch.bfloat16, BS=1, seed=34)
    out, lse = _run(p)
    rows = list(p.refs(0.125, True, out.dtype))
    for i in (0, 1, 1000, n - 2, n - 1):
        q0, nq, ref = rows[i]
        po.check(out[q0:q0 + nq], lse[:, q0:q0 + nq], ref, f"row {i}")
    again = _run(p)
    assert torch.equal(out, again[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("qs,ks", [([40] * 30, [6500] * 2 + [9] * 28), ([3], [6500])], ids=["chunks", "one"])
def test_tables_as_long_as_they_get(gpu, dtype, D, qs, ks):
    """Single-token blocks, a place looked up for every key, beside the largest stages."""
    qs = [min(q, k) for q, k in zip(qs, ks)]
    p = po.Paged(qs, ks, 16, 16, D, dtype, BS=1, seed=36)
    out, lse = _run(p)
    rows = [(0, 0), (sum(qs[:-1]), len(qs) - 1)]
    for q0, i in rows:
        for h in (0, 15):
            q = p.q[q0:q0 + qs[i], h:h + 1]
            ref = po.attend(q, p.k[i][:, h:h + 1], p.v[i][:, h:h + 1], 0.125, True, out.dtype)
            po.check(out[q0:q0 + qs[i], h:h + 1], lse[h:h + 1, q0:q0 + qs[i]], ref, f"row {i} head {h}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_arrival_counters(gpu, dtype, monkeypatch):
    """A caller that gives no counters: they lie in the workspace, and a graph clears them."""
    monkeypatch.setattr(ops, "_counters_ptr", lambda *a, **k: None)
    p = po.Paged([70, 3], [3000, 1200], 4, 2, 64, dtype, seed=35)
    args = dict(kv=p.kv.to(gpu), q=p.q.to(gpu), bt=p.bt.to(gpu), cu=p.cu.to(gpu), ln=p.lens.to(gpu))

    def call():
        return ops.paged_prefill(args["q"], args["kv"][..., :64], args["kv"][..., 64:], args["bt"],
                                 args["cu"], args["ln"], 0.125, max_seqlen_q=70, max_seqlen_k=3000)

    eager = call()
    _check(p, *eager)
    side = torch.cuda.Stream()
    ops.reserve_workspace(side, 1 << 26)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        call()
    ops.release_workspace(side)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 72])
def test_a_cache_in_pinned_host_memory(gpu, dtype, D):
    """The host tier's own layout, read in place."""
    p = po.Paged([40, 2], [300, 900], 4, 2, D, dtype, seed=37)
    k, v = (pinned_zeros((p.B, 2, p.BS, D), dtype) for _ in range(2))
    k.copy_(p.kv[..., :D].transpose(1, 2))
    v.copy_(p.kv[..., D:].transpose(1, 2))
    _check(p, *_run(p, k=k.transpose(1, 2), v=v.transpose(1, 2)))


def test_output_over_the_queries(gpu):
    """Every tile reads its own queries only, and before it writes."""
    p = po.Paged([130, 3], [2000, 1000], 8, 2, 64, torch.bfloat16, seed=38)
    kv, q = p.kv.to(gpu), p.q.to(gpu)
    ops.paged_prefill(q, kv[..., :64], kv[..., 64:], p.bt.to(gpu), p.cu.to(gpu), p.lens.to(gpu),
                      0.125, max_seqlen_q=130, max_seqlen_k=2000, out=q)
    out, _ = _run(p)
    assert torch.equal(q, out)


def test_two_streams_at_once(gpu):
    """Divided calls on two streams, each with its own scratch and counters."""
    ps = [po.Paged([60, 2], [2500, 3000], 8, 2, 64, torch.float16, seed=s) for s in (39, 40)]
    dev = [dict(q=p.q.to(gpu), kv=p.kv.to(gpu), bt=p.bt.to(gpu), cu=p.cu.to(gpu), ln=p.lens.to(gpu))
           for p in ps]
    want = [_run(p) for p in ps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for x, s, g in zip(dev, streams, got):
            with torch.cuda.stream(s):
                g.append(ops.paged_prefill(x["q"], x["kv"][..., :64], x["kv"][..., 64:], x["bt"],
                                           x["cu"], x["ln"], 0.125, 60, 3000))
    torch.cuda.synchronize()
    for g, (out, lse) in zip(got, want):
        for o, l in g:
            assert torch.equal(o, out) and torch.equal(l, lse)


@pytest.mark.parametrize("D", [128, 256, 72])
def test_cache_offsets_past_32_bits(gpu, D):
    """Blocks at the far end of a cache of more than 2^31 elements: the same bits as at its start."""
    p = po.Paged([130, 2], [700, 400], 4, 2, D, torch.bfloat16, seed=44)
    kv = p.kv.to(gpu)
    elements = p.BS * 2 * 2 * D
    far = 2 ** 31 // elements + 5
    big = torch.empty(far + p.B, p.BS, 2, 2 * D, dtype=torch.bfloat16, device=gpu)
    big[far:] = kv
    want = _run(p)
    bt = torch.where(p.bt >= 0, p.bt + far, p.bt)
    got = _run(p, k=big[..., :D], v=big[..., D:], bt=bt)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(p, *got)
