"""The native calls of paged_prefill, varlen_attention and build_tables against the same calls
through ctypes: results, outputs given, refusals, graphs."""

from __future__ import annotations

import pytest
import torch

from tests import prefill_oracle as po
from vllm_fastdecoder_amd import ops

pytestmark = pytest.mark.gpu


@pytest.fixture
def native(gpu):
    mod = ops._native()
    if not mod:
        pytest.skip("no native call module")
    return mod


def _both(monkeypatch, call):
    here = call()
    monkeypatch.setattr(ops, "_NATIVE", False)
    monkeypatch.setattr(ops, "_native", lambda: False)
    there = call()
    monkeypatch.undo()
    for a, b in zip(here, there):
        if a is None:
            assert b is None
        else:
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
            assert torch.equal(a, b)
    return here


class _Only:
    """A native module whose calls must be taken here."""

    def __init__(self, mod, name):
        def call(*a):
            got = getattr(mod, name)(*a)
            assert got is not None, f"{name} went through ctypes"
            self.calls += 1
            return got

        self.calls = 0
        setattr(self, name, call)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qs,ks", [([5], [900]), ([3, 120, 1], [40, 700, 2500])], ids=str)
def test_paged(gpu, native, monkeypatch, dtype, qs, ks):
    p = po.Paged(qs, ks, 8, 2, 64, dtype, seed=41, extra_cols=40)
    kv, q, bt, cu, ln = (x.to(gpu) for x in (p.kv, p.q, p.bt, p.cu, p.lens))
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    for qq in (q, turned):
        for out_dtype in (None, torch.float32):
            for longest in (None, max(ks)):
                def call(mod=None):
                    out = None if out_dtype is None else torch.zeros(q.shape, dtype=out_dtype, device=gpu)
                    return ops.paged_prefill(qq, kv[..., :64], kv[..., 64:], bt, cu, ln, 0.125,
                                             max_seqlen_q=max(qs), max_seqlen_k=longest, out=out)

                _both(monkeypatch, call)
                only = _Only(native, "paged_prefill")
                monkeypatch.setattr(ops, "_NATIVE", only)
                call()
                monkeypatch.undo()
                assert only.calls == 1


@pytest.mark.parametrize("causal", [True, False])
def test_packed(gpu, native, monkeypatch, causal):
    g = torch.Generator(device="cuda").manual_seed(42)
    qkv = torch.randn(300, 12, 64, generator=g, device=gpu).to(torch.bfloat16)
    cu = torch.tensor([0, 100, 100, 260], dtype=torch.int32, device=gpu)

    def call():
        return ops.varlen_attention(qkv[:260, :8], qkv[:, 8:10], qkv[:, 10:], cu, cu, 0.125, 160,
                                    160, causal=causal)

    _both(monkeypatch, call)
    only = _Only(native, "varlen_attention")
    monkeypatch.setattr(ops, "_NATIVE", only)
    call()
    assert only.calls == 1


@pytest.mark.parametrize("taking", [True, False])
def test_tables(gpu, native, monkeypatch, taking):
    qsl = torch.tensor([0, 5, 6, 40], dtype=torch.int32, device=gpu)
    ctx = torch.tensor([11, 64, 0], dtype=torch.int32, device=gpu)
    free = torch.arange(30, 60, dtype=torch.int32, device=gpu)
    start = torch.arange(30, dtype=torch.int32, device=gpu).reshape(3, 10)
    errors = torch.zeros(1, dtype=torch.int32, device=gpu)

    def call():
        bt = start.clone()
        taken = torch.full((1,), 2, dtype=torch.int32, device=gpu)
        got = ops.build_tables(qsl, ctx, bt, 16, 44, 60, free_blocks=free if taking else None,
                               taken=taken if taking else None, error_count=errors)
        return got + (bt,)

    _both(monkeypatch, call)
    only = _Only(native, "build_tables")
    monkeypatch.setattr(ops, "_NATIVE", only)
    call()
    assert only.calls == 1 and int(errors) == 0


def test_refusals_are_the_checks_own(gpu, native):
    """What the native call does not take is refused with the same words as ever."""
    kc = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=gpu)
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device=gpu)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=gpu)
    bt = torch.zeros(1, 4, dtype=torch.int32, device=gpu)
    ln = torch.tensor([3], dtype=torch.int32, device=gpu)
    with pytest.raises(RuntimeError, match="num_heads"):
        ops.paged_prefill(q[:, :3], kc, kc, bt, cu, ln, 1.0, 3)
    with pytest.raises(RuntimeError, match="int32"):
        ops.paged_prefill(q, kc, kc, bt.long(), cu, ln, 1.0, 3)
    with pytest.raises(RuntimeError, match="max_seqlen_q"):
        ops.varlen_attention(q, q, q, cu, cu, 1.0, -1, 3)
    with pytest.raises(RuntimeError, match="block_size"):
        ops.build_tables(cu, ln, bt, 0, 3, 4)
    with pytest.raises(RuntimeError, match="together"):
        ops.build_tables(cu, ln, bt, 16, 3, 4, free_blocks=ln)


def test_captured(gpu, native):
    """Native calls of a whole step in one graph: tables, attention of a chunk, fresh rows."""
    p = po.Paged([70, 2], [1500, 900], 8, 2, 64, torch.bfloat16, seed=43)
    kv, q, bt, cu, ln = (x.to(gpu) for x in (p.kv, p.q, p.bt, p.cu, p.lens))
    ctx = ln - (cu[1:] - cu[:-1])
    k, v = q[:, :2].contiguous(), q[:, 2:4].contiguous()

    def step():
        slots, pos, lens, _ = ops.build_tables(cu, ctx, bt, 16, p.T, p.B)
        a, _ = ops.paged_prefill(q, kv[..., :64], kv[..., 64:], bt, cu, lens, 0.125, 70, 1500)
        b, _ = ops.varlen_attention(q, k, v, cu, cu, 0.125, 70, 70, causal=True)
        return slots, pos, lens, a, b

    eager = step()
    assert torch.equal(eager[2], ln)
    side = torch.cuda.Stream()
    ops.reserve_workspace(side, 1 << 26)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, eager):
            assert torch.equal(x, y)
        step()
    ops.release_workspace(side)
