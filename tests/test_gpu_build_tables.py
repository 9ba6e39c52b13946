"""GPU checks of build_tables against a plain host restatement, value for value."""

from __future__ import annotations

import pytest
import torch

from tests import prefill_oracle as po
from vllm_fastdecoder_amd import ops

pytestmark = pytest.mark.gpu


def _host(qsl, ctx, bt, BS, T, num_blocks, free, taken):
    """The operator row by row: (slots, positions, lens, taken, table, errors)."""
    bt = bt.clone()
    W = bt.shape[1]
    slots, pos = [-1] * T, [0] * T
    lens, errors = [], 0
    at = used = taken if free is not None else 0
    for r in range(len(ctx)):
        q0, q1, c = int(qsl[r]), int(qsl[r + 1]), int(ctx[r])
        L = c + q1 - q0
        lens.append(L)
        ok = 0 <= q0 <= q1 <= T and c >= 0 and L <= W * BS
        if ok and free is not None:
            held, need = -(-c // BS), -(-L // BS) - -(-c // BS)
            if need and (taken < 0 or at + need > len(free)):
                ok = False
            else:
                for k in range(need):
                    bt[r, held + k] = free[at + k]
                used += need
            at += need
        errors += not ok
        for t in range(max(q0, 0), min(q1, T)):
            pos[t] = c + t - q0
            if ok:
                b = int(bt[r, pos[t] // BS])
                if 0 <= b < num_blocks:
                    slots[t] = b * BS + pos[t] % BS
                else:
                    errors += 1
    return slots, pos, lens, used, bt, errors


def _check(gpu, qs, ctx, BS, W, pad=0, free_len=None, taken=0, num_blocks=None, seed=0,
           alloc=True, qsl=None):
    g = torch.Generator().manual_seed(seed)
    n = len(ctx)
    qsl = po.starts(qs) if qsl is None else torch.tensor(qsl, dtype=torch.int32)
    T = sum(qs) + pad
    bt = torch.randint(0, 5000, (n, W), generator=g, dtype=torch.int32)
    num_blocks = 5000 if num_blocks is None else num_blocks
    free = torch.randperm(5000, generator=g)[:free_len if free_len is not None else 4000].int()
    ctx_t = torch.tensor(ctx, dtype=torch.int32)
    want = _host(qsl, ctx, bt, BS, T, num_blocks, free if alloc else None, taken)
    table = bt.to(gpu)
    wide = torch.full((n, W + 3), -3, dtype=torch.int32, device=gpu)
    wide[:, 1:W + 1] = table
    for view in (table, wide[:, 1:W + 1]):
        for _ in range(2):  # the same call again changes nothing
            err = torch.zeros(1, dtype=torch.int32, device=gpu)
            tk = torch.tensor([taken], dtype=torch.int32, device=gpu)
            slots, pos, lens, out = ops.build_tables(
                qsl.to(gpu), ctx_t.to(gpu), view, BS, T, num_blocks,
                free_blocks=free.to(gpu) if alloc else None, taken=tk if alloc else None,
                error_count=err)
            assert slots.tolist() == want[0]
            assert pos.tolist() == want[1]
            assert lens.tolist() == want[2]
            assert torch.equal(view.cpu(), want[4])
            assert int(err) == want[5]
            if alloc:
                assert int(out) == want[3] and int(tk) == taken
            else:
                assert out is None
    assert torch.all(wide[:, 0] == -3) and torch.all(wide[:, W + 1:] == -3)


@pytest.mark.parametrize("BS", [1, 16, 24, 64])
@pytest.mark.parametrize("alloc", [True, False])
@pytest.mark.parametrize("n,qmax,cmax", [(1, 1, 50), (1, 700, 0), (5, 40, 300), (64, 1, 900),
                                         (256, 1, 500), (300, 9, 60), (1100, 2, 30), (700, 0, 9)])
def test_steps(gpu, n, qmax, cmax, BS, alloc):
    import random

    rng = random.Random(n * 7 + qmax + BS)
    qs = [rng.randint(0, qmax) if rng.random() < 0.3 else qmax for _ in range(n)]
    ctx = [rng.randint(0, cmax) for _ in range(n)]
    W = max(-(-(c + q) // BS) for c, q in zip(ctx, qs)) + 2
    _check(gpu, qs, ctx, BS, W, pad=rng.choice((0, 5)), taken=rng.choice((0, 7)), alloc=alloc,
           seed=n)


def test_free_list_ends(gpu):
    """Rows take in order; those behind the end of the list get nothing, rows that need no block
    still get their slots."""
    qs, ctx = [20, 1, 100, 1, 16, 5], [0, 3, 8, 16, 0, 1]
    for free_len in range(0, 14):
        _check(gpu, qs, ctx, 16, 9, free_len=free_len, taken=0)
        _check(gpu, qs, ctx, 16, 9, free_len=free_len, taken=2)
    _check(gpu, [300] * 300, [0] * 300, 16, 19, free_len=4000)  # ends in the second group of rows
    _check(gpu, qs, ctx, 16, 9, taken=-1)


def test_bad_rows_and_ids(gpu):
    """Rows too long for the table, of negative length or whose tokens do not lie in the step, and
    ids past the caches: counted, no block taken, no slot."""
    _check(gpu, [5, 200, 7], [10, 0, 3], 16, 4)
    _check(gpu, [5, 2, 7], [10, -4, 3], 16, 4)
    _check(gpu, [5, 2, 7], [10, 4, 3], 16, 4, num_blocks=2500)
    _check(gpu, [5, 2, 7], [10, 4, 3], 16, 4, num_blocks=2500, alloc=False)
    _check(gpu, [5, 2, 7], [10, 4, 3], 16, 4, qsl=[0, 5, 7, 90])


def test_no_rows_and_no_tokens(gpu):
    _check(gpu, [], [], 16, 4, pad=9)
    _check(gpu, [], [], 16, 4, taken=3)
    _check(gpu, [0, 0], [16, 3], 16, 4)
    _check(gpu, [3, 0], [16, 3], 16, 0, pad=1)


def test_captured(gpu):
    qs, ctx = [1] * 40, list(range(10, 50))
    bt = torch.zeros(40, 8, dtype=torch.int32, device=gpu)
    free = torch.arange(1000, dtype=torch.int32, device=gpu).flip(0).contiguous()
    qsl, c = po.starts(qs).to(gpu), torch.tensor(ctx, dtype=torch.int32, device=gpu)
    taken = torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.build_tables(qsl, c, bt.clone(), 16, 40, 1000, free_blocks=free, taken=taken)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.build_tables(qsl, c, bt, 16, 40, 1000, free_blocks=free, taken=taken)
        taken.copy_(got[3])
        c.add_(1)
    host_bt, host_taken, host_c = bt.cpu(), 0, list(ctx)
    for _ in range(20):  # twenty decode steps, their tables kept on the GPU
        graph.replay()
        want = _host(po.starts(qs), host_c, host_bt, 16, 40, 1000, free.cpu(), host_taken)
        torch.cuda.synchronize()
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
        assert torch.equal(bt.cpu(), want[4]) and int(taken) == want[3]
        host_bt, host_taken, host_c = want[4], want[3], [x + 1 for x in host_c]
