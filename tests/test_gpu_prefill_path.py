"""The step operators together, as a serving step uses them: tables from lengths, the cache write,
and attention of decodes, chunks and fresh prompts, through the package's own orchestration and by
themselves."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch

from tests import prefill_oracle as po
from tests.test_gpu_forward import REQS16, TOL, build_tiers
from vllm_fastdecoder_amd import backend, ops, plan, state

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _store():
    yield
    state.STORE = None


# REQS16 with a chunk of a prompt with context, all its blocks in HBM (a P row of many tokens)
REQS = REQS16 + [(37, 70, [13, 14, 15, 16, 17, 18, 19])]


@pytest.mark.parametrize("H,KVH", [(4, 4), (8, 2)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_split_step_without_another_attention(gpu, H, KVH, dtype):
    """_forward_split with the library's own ops: S, P and F rows."""
    G, C, BS, D = 24, 40, 16, 128
    sc = build_tiers(REQS, G, C, H, KVH, D, BS, dtype, 1, gpu)
    hp = plan.build_host_plan(sc.qsl, sc.seq, sc.bt, sc.slots, G, C, BS)
    dp = plan.to_device(hp, sc.bt.to(gpu), gpu)
    assert hp.p_max_q == 70 and hp.n_f_tok
    state.STORE = state.HostKVStore(G, C, BS, KVH, D, dtype, k={"l0": sc.host_k},
                                    v={"l0": sc.host_v})
    assert backend.make_ops() is backend.HipOps is backend.OPS
    impl = backend.SplitDecodeImpl(H, KVH, D, sc.scale, cpu_fraction=0.0)
    out = torch.full_like(sc.query, math.nan)
    impl._forward_split(SimpleNamespace(layer_name="l0"), sc.query, sc.key, sc.value, sc.kv_cache,
                        dp, out)
    torch.cuda.synchronize()
    assert float((out.double().cpu() - sc.ref).abs().max()) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_step_planned_on_the_gpu_from_its_lengths(gpu, dtype):
    """build_device_step without a slot mapping: decodes in both tiers and fresh prompts."""
    G, C, BS, D, H, KVH = 24, 40, 16, 128, 8, 2
    sc = build_tiers(REQS16, G, C, H, KVH, D, BS, dtype, 2, gpu)
    state.STORE = state.HostKVStore(G, C, BS, KVH, D, dtype, k={"l0": sc.host_k},
                                    v={"l0": sc.host_v})
    R = len(REQS16)
    step = backend.build_device_step(sc.qsl, sc.seq, sc.bt.to(gpu), None, R, state.STORE, gpu)
    given = backend.build_device_step(sc.qsl, sc.seq, sc.bt.to(gpu), sc.slots.to(gpu), R,
                                      state.STORE, gpu)
    assert torch.equal(step.gpu_slots, given.gpu_slots)
    assert torch.equal(step.host_slots, given.host_slots)
    impl = backend.SplitDecodeImpl(H, KVH, D, sc.scale, cpu_fraction=0.0)
    out = torch.full_like(sc.query, math.nan)
    impl._forward_device(SimpleNamespace(layer_name="l0"), sc.query, sc.key, sc.value, sc.kv_cache,
                         step, out)
    step.check_errors()
    assert float((out.double().cpu() - sc.ref).abs().max()) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_prompts_in_chunks(gpu, dtype):
    """Three requests served from their lengths alone: each step's blocks and slots are made on the
    GPU, its K and V written, its tokens attended; every step against the whole history."""
    H, KVH, D, BS, B = 8, 2, 64, 16, 80
    scale = 1 / math.sqrt(D)
    g = torch.Generator().manual_seed(0)
    kv = torch.full((B, BS, KVH, 2 * D), math.nan, dtype=dtype, device=gpu)
    bt = torch.zeros(3, 40, dtype=torch.int32, device=gpu)
    free = torch.randperm(B, generator=g).int().to(gpu)
    taken = torch.zeros(1, dtype=torch.int32, device=gpu)
    hist_k = [torch.empty(0, KVH, D, dtype=dtype) for _ in range(3)]
    hist_v = [torch.empty(0, KVH, D, dtype=dtype) for _ in range(3)]
    errors = torch.zeros(1, dtype=torch.int32, device=gpu)
    for qs in ([200, 1, 0], [90, 60, 5], [1, 1, 1], [1, 150, 1], [16, 1, 30], [1, 1, 1]):
        T = sum(qs)
        q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (H, KVH, KVH))
        cu = po.starts(qs)
        ctx = torch.tensor([x.shape[0] for x in hist_k], dtype=torch.int32)
        slots, pos, lens, taken = ops.build_tables(cu.to(gpu), ctx.to(gpu), bt, BS, T + 3, B,
                                                   free_blocks=free, taken=taken,
                                                   error_count=errors)
        pad = torch.zeros(3, KVH, D, dtype=dtype)
        ops.reshape_and_cache(torch.cat([k, pad]).to(gpu), torch.cat([v, pad]).to(gpu),
                              kv[..., :D], kv[..., D:], slots)
        out, lse = backend.HipOps.fa(q=q.to(gpu), k=kv[..., :D], v=kv[..., D:],
                                     cu_seqlens_q=cu.to(gpu), max_seqlen_q=max(qs),
                                     seqused_k=lens, max_seqlen_k=int(ctx.max()) + max(qs),
                                     softmax_scale=scale, causal=True, block_table=bt,
                                     return_softmax_lse=True, window_size=(-1, -1))
        fresh, _ = ops.varlen_attention(q.to(gpu), k.to(gpu), v.to(gpu), cu.to(gpu), cu.to(gpu),
                                        scale, max(qs), max(qs), causal=True)
        for i in range(3):
            q0, q1 = int(cu[i]), int(cu[i + 1])
            hist_k[i] = torch.cat([hist_k[i], k[q0:q1]])
            hist_v[i] = torch.cat([hist_v[i], v[q0:q1]])
            po.check(out[q0:q1], lse[:, q0:q1],
                     po.attend(q[q0:q1], hist_k[i], hist_v[i], scale, True, dtype), f"request {i}")
            if int(ctx[i]) == 0:  # without context the cache holds just the step's own
                ref = po.attend(q[q0:q1], k[q0:q1], v[q0:q1], scale, True, dtype)[0]
                assert float((fresh[q0:q1].double().cpu() - ref).abs().max() if q1 > q0 else 0) \
                    <= TOL[dtype]
    assert int(errors) == 0 and int(taken) == sum(-(-x.shape[0] // BS) for x in hist_k)


def test_forms_that_fa_refuses(gpu):
    q = torch.zeros(4, 4, 64, dtype=torch.float16, device=gpu)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=gpu)
    form = dict(q=q, k=q, v=q, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=4, max_seqlen_k=4,
                softmax_scale=0.1, causal=True)
    assert backend.HipOps.fa(**form).shape == q.shape
    for bad in (dict(softcap=20.0), dict(window_size=(128, 0)), dict(cu_seqlens_k=None),
                dict(cu_seqlens_q=None), dict(alibi_slopes=torch.zeros(4)),
                dict(block_table=cu[None])):
        with pytest.raises(NotImplementedError):
            backend.HipOps.fa(**{**form, **bad})
