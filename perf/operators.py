"""Timed work of the step operators around decode: prompts, chunks of prompts and their tables.

Every case is one call of the package's public entry points on inputs already
on the GPU (`own` true), or the same operator written out in elementary torch
operations in 32 bits (`own` false):

  chunk   ops.paged_prefill: the attention of one layer for a step whose rows
          bring several new tokens each (a chunk of a prompt, tokens to verify)
          or one (`singles` rows: decodes in the same step) over the paged HBM
          cache, in which the new tokens' K and V already lie. Token j of a row
          of q new tokens and L tokens in all sees keys 0 .. L - q + j.
  fresh   ops.varlen_attention: attention over the step's own packed K and V,
          without a cache: prompts without context (causal), or a decoder's
          tokens over the states of an encoder of another length (not causal).
  tables  ops.build_tables: a step's new cache blocks, slot mapping, positions
          and sequence lengths, from its requests' lengths.

Lengths depend on the case alone (so its work is known without its inputs);
the seed decides which row has which length, where the blocks lie, and the
values, N(0, 1) as in the repository's workloads.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# (query heads, kv heads, head size): the decode cases' layouts
LAYOUTS = ((32, 32, 128), (32, 8, 128), (28, 4, 128), (8, 1, 128), (16, 8, 256), (32, 32, 80),
           (32, 32, 64), (14, 2, 64), (16, 2, 96), (40, 8, 128))
LARGEST_FLOPS = 2.1e12    # the long chunk below
LARGEST_SCORES = 4.4e9    # and its scores, as the plain form holds them


def _chunk(name, n, q, ctx, heads, dtype, bs=16, singles=0, capacity=0):
    H, KVH, D = heads
    return {"name": name, "kind": "chunk", "n": n, "q_lo": q[0], "q_hi": q[1], "c_lo": ctx[0],
            "c_hi": ctx[1], "singles": singles, "H": H, "KVH": KVH, "D": D, "BS": bs,
            "dtype": dtype, "capacity": capacity}


def _fresh(name, n, q, k, heads, dtype, causal):
    H, KVH, D = heads
    return {"name": name, "kind": "fresh", "n": n, "q_lo": q[0], "q_hi": q[1], "k_lo": k[0],
            "k_hi": k[1], "H": H, "KVH": KVH, "D": D, "dtype": dtype, "causal": causal}


def listed() -> list[dict]:
    return [
        # one interactive user, five tokens to verify: the smallest call, where latency counts
        _chunk("chunk_verify_one", 1, (5, 5), (900, 900), (32, 8, 128), "bf16", capacity=8192),
        # a batch of requests with a few tokens to verify each, contexts from new to long
        _chunk("chunk_verify_batch", 48, (2, 9), (50, 3100), (28, 4, 128), "bf16", bs=32,
               capacity=8192),
        # chunks of a few prompts (the scheduler's token budget of about 2048)
        _chunk("chunk_prompts", 4, (389, 640), (256, 2048), (32, 8, 128), "bf16"),
        # a serving step: decodes and one chunk of a prompt in one call, multi-head
        _chunk("chunk_mixed_step", 32, (500, 500), (128, 1024), (32, 32, 128), "fp16", singles=31),
        # a long document's last chunk
        _chunk("chunk_long_document", 1, (4096, 4096), (28_000, 28_000), (32, 8, 128), "bf16"),
        # head size 256, two query heads per kv head
        _chunk("chunk_head_256", 3, (200, 700), (200, 4000), (16, 8, 256), "bf16"),
        # fp32 caches, the repository's third data type
        _chunk("chunk_fp32", 3, (100, 300), (64, 1500), (32, 8, 128), "fp32"),
        # fresh prompts of a multi-head model (the repository's simulation: 64 to 512 tokens)
        _fresh("fresh_prompts", 16, (64, 512), (0, 0), (32, 32, 128), "fp16", True),
        # one long fresh prompt of a grouped-query model
        _fresh("fresh_long_prompt", 1, (8192, 8192), (0, 0), (32, 8, 128), "bf16", True),
        # cross attention: decoders' tokens over an encoder's states, head size 64
        _fresh("cross_encoder", 6, (30, 448), (1500, 1500), (20, 20, 64), "fp16", False),
        # a decode step's tables: one new token per request, now and then a new block
        {"name": "tables_decode", "kind": "tables", "n": 256, "q_lo": 1, "q_hi": 1, "c_lo": 1024,
         "c_hi": 4096, "BS": 16, "capacity": 8192, "pad": 0},
        # the tables of a step of many prompts, the token count padded for a captured graph
        {"name": "tables_prompts", "kind": "tables", "n": 67, "q_lo": 64, "q_hi": 512, "c_lo": 0,
         "c_hi": 700, "BS": 16, "capacity": 2048, "pad": 77},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    """Another case of the same ranges: mostly attention, sizes spread over their logarithm."""
    while True:
        pick = rng.random()
        if pick < 0.15:
            q = _log_int(rng, 1, 512)
            return {"kind": "tables", "n": _log_int(rng, 1, 512), "q_lo": 1, "q_hi": q,
                    "c_lo": 0, "c_hi": _log_int(rng, 16, 6000), "BS": rng.choice((16, 32, 64)),
                    "capacity": 8192, "pad": rng.choice((0, 0, rng.randrange(1, 100)))}
        H, KVH, D = rng.choice(LAYOUTS)
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        q = _log_int(rng, 1, 8192)
        q_lo = max(1, q - int(q * rng.choice((0.0, 0.5, 0.9))))
        if pick < 0.7:
            c = _log_int(rng, 16, 32_000)
            c_lo = c - int(c * rng.choice((0.0, 0.5, 1.0)))
            n = _log_int(rng, 1, 64)
            case = {"kind": "chunk", "n": n, "q_lo": q_lo, "q_hi": q, "c_lo": c_lo, "c_hi": c,
                    "singles": rng.choice((0, 0, n // 2)), "H": H, "KVH": KVH, "D": D,
                    "BS": rng.choice((16, 32, 64)), "dtype": dtype,
                    "capacity": rng.choice((0, 0, 65_536))}
        else:
            k = _log_int(rng, 1, 8192)
            causal = rng.random() < 0.6
            case = {"kind": "fresh", "n": _log_int(rng, 1, 64), "q_lo": q_lo, "q_hi": q,
                    "k_lo": 0 if causal else max(1, k // 2), "k_hi": 0 if causal else k, "H": H,
                    "KVH": KVH, "D": D, "dtype": dtype, "causal": causal}
        qs, ks = _lens(case)
        padded = case["n"] * H * max(qs) * max(ks)
        if padded <= LARGEST_SCORES and work(case)["flops"] <= LARGEST_FLOPS:
            return case


# ------------------------------------------------------------------ inputs


def _blocks(tokens: int, bs: int) -> int:
    return -(-tokens // bs)


def _lens(case) -> tuple[list[int], list[int]]:
    """Each row's new tokens and keys, a function of the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    qs = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n"])]
    if case["kind"] == "fresh":
        ks = qs if case["causal"] else [rng.randint(case["k_lo"], case["k_hi"]) for _ in qs]
        return qs, list(ks)
    for i in range(case.get("singles", 0)):
        qs[i] = 1
    return qs, [q + rng.randint(case["c_lo"], case["c_hi"]) for q in qs]


class _Draws:
    """Seeded values: small things on the CPU, the rest straight on the GPU."""

    def __init__(self, seed: int):
        self.cpu = torch.Generator().manual_seed(seed)
        self.gpu = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype) -> torch.Tensor:
        return torch.randn(shape, generator=self.gpu, device="cuda").to(dtype)

    def perm(self, n: int) -> list[int]:
        return torch.randperm(n, generator=self.cpu).tolist()

    def tables(self, counts: list[int], width: int, pool: int):
        """Each row's blocks: distinct ids scattered over the pool; and the ids left over."""
        ids = torch.randperm(pool, generator=self.cpu).to(torch.int32)
        bt = torch.zeros(len(counts), max(width, 1), dtype=torch.int32)
        pos = 0
        for i, c in enumerate(counts):
            bt[i, :c] = ids[pos:pos + c]
            pos += c
        return bt, ids[pos:].contiguous()


def _starts(lens: list[int]) -> torch.Tensor:
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)


def prepare(case, seed):
    draws = _Draws(seed)
    qs, ks = _lens(case)
    order = draws.perm(case["n"])
    qs, ks = [qs[i] for i in order], [ks[i] for i in order]
    st = {"case": case, "qs": qs, "ks": ks, "max_q": max(qs), "max_k": max(ks),
          "cu_q": _starts(qs).cuda(), "T": sum(qs)}
    if case["kind"] == "tables":
        bs = case["BS"]
        ctx = [k - q for q, k in zip(qs, ks)]
        held = [_blocks(c, bs) for c in ctx]
        pool = sum(_blocks(k, bs) for k in ks) + 100
        bt, free = draws.tables(held, _blocks(max(case["capacity"], max(ks)), bs), pool)
        st.update(ctx=torch.tensor(ctx, dtype=torch.int32).cuda(), bt=bt.cuda(), free=free.cuda(),
                  taken=torch.full((1,), 3, dtype=torch.int32, device="cuda"), pool=pool,
                  T=sum(qs) + case["pad"])
        return st
    dt, H, KVH, D = DTYPES[case["dtype"]], case["H"], case["KVH"], case["D"]
    st["q"] = draws.normal((sum(qs), H, D), dt)
    if case["kind"] == "fresh":
        st["k"] = draws.normal((sum(ks), KVH, D), dt)
        st["v"] = draws.normal((sum(ks), KVH, D), dt)
        st["cu_k"] = st["cu_q"] if case["causal"] else _starts(ks).cuda()
        return st
    bs = case["BS"]
    counts = [_blocks(k, bs) for k in ks]
    bt, _ = draws.tables(counts, _blocks(max(case["capacity"], max(ks)), bs), sum(counts))
    kv = draws.normal((sum(counts), bs, KVH, 2 * D), dt)
    st.update(k=kv[..., :D], v=kv[..., D:], bt=bt.cuda(),
              lens=torch.tensor(ks, dtype=torch.int32).cuda())
    return st


# ------------------------------------------------------------------ one pass


def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from vllm_fastdecoder_amd import ops

        if kind == "tables":
            return ops.build_tables(st["cu_q"], st["ctx"], st["bt"], case["BS"], st["T"],
                                    st["pool"], free_blocks=st["free"],
                                    taken=st["taken"]) + (st["bt"],)
        scale = 1.0 / math.sqrt(case["D"])
        if kind == "chunk":
            return ops.paged_prefill(st["q"], st["k"], st["v"], st["bt"], st["cu_q"], st["lens"],
                                     scale, max_seqlen_q=st["max_q"], max_seqlen_k=st["max_k"])
        return ops.varlen_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], scale,
                                    max_seqlen_q=st["max_q"], max_seqlen_k=st["max_k"],
                                    causal=case["causal"])
    if kind == "tables":
        return _plain_tables(st, case["BS"])
    if kind == "chunk":
        cols = _blocks(st["max_k"], case["BS"])
        ids = st["bt"][:, :cols].long()
        k, v = st["k"][ids].flatten(1, 2), st["v"][ids].flatten(1, 2)  # [n, keys, KVH, D]
        return _plain_attention(st, k, v, st["lens"], True)
    starts = st["cu_k"].long()
    at = starts[:-1, None] + torch.arange(st["max_k"], device=starts.device)
    at.clamp_(max=st["k"].shape[0] - 1)
    return _plain_attention(st, st["k"][at], st["v"][at], st["cu_k"].diff(), case["causal"])


def _plain_attention(st, k, v, lens, causal):
    """Rows padded to the longest, k and v [n, keys, KVH, D] -> out [T, H, D], lse [H, T]."""
    q, starts = st["q"], st["cu_q"].long()
    T, H, D = q.shape
    n, L, KVH, _ = k.shape
    M, G, dev = st["max_q"], H // KVH, q.device
    new = starts.diff()
    at = (starts[:-1, None] + torch.arange(M, device=dev)).clamp_(max=T - 1)
    qp = q[at].float().view(n, M, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(n, KVH, G * M, D)
    s = torch.matmul(qp, k.permute(0, 2, 3, 1).float().contiguous())
    s = s.view(n, KVH, G, M, L).mul_(1.0 / math.sqrt(D))
    key = torch.arange(L, device=dev)
    last = lens.long()[:, None] - 1  # the last key that a token sees
    if causal:
        last = last - new[:, None] + 1 + torch.arange(M, device=dev)
    last = torch.minimum(last, lens.long()[:, None] - 1)
    s.masked_fill_((key > last[..., None])[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, KVH, G * M, L), v.permute(0, 2, 1, 3).float().contiguous())
    o = o.view(n, KVH, G, M, D) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + total.log()).squeeze(-1)
    tok = torch.arange(T, device=dev)
    row = torch.searchsorted(starts, tok, right=True) - 1
    j = tok - starts[row]
    out = o.permute(0, 3, 1, 2, 4)[row, j].reshape(T, H, D).to(q.dtype)
    return out, lse.permute(0, 3, 1, 2)[row, j].reshape(T, H).t().contiguous()


def _plain_tables(st, bs):
    starts, ctx, bt, free = st["cu_q"].long(), st["ctx"].long(), st["bt"], st["free"]
    n, W = bt.shape
    dev = bt.device
    lens = ctx + starts.diff()
    held = (ctx + bs - 1) // bs
    need = (lens + bs - 1) // bs - held
    first = st["taken"].long() + need.cumsum(0) - need
    col = torch.arange(W, device=dev)
    k = col - held[:, None]
    fresh = free[(first[:, None] + k).clamp_(0, free.shape[0] - 1)]
    bt.copy_(torch.where((k >= 0) & (k < need[:, None]), fresh, bt))
    tok = torch.arange(st["T"], device=dev)
    row = (torch.searchsorted(starts, tok, right=True) - 1).clamp_(max=n - 1)
    pos = ctx[row] + tok - starts[row]
    real = tok < starts[-1]
    pos = torch.where(real, pos, torch.zeros_like(pos))
    slot = bt[row, (pos // bs).clamp_(max=W - 1)].long() * bs + pos % bs
    slot = torch.where(real, slot, torch.full_like(slot, -1))
    taken = st["taken"] + need.sum().to(torch.int32)
    return slot, pos, lens.to(torch.int32), taken, bt


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    """Attention: q, out and lse, every row's keys and values, ids and lengths, each once; a
    product with K and one with V per query token, head and key it sees. Tables: the ids that
    change and the per-token and per-request values."""
    qs, ks = _lens(case)
    n, T = case["n"], sum(qs)
    if case["kind"] == "tables":
        bs = case["BS"]
        new = sum(_blocks(k, bs) - _blocks(k - q, bs) for q, k in zip(qs, ks))
        used = sum(_blocks(k, bs) - (k - q) // bs for q, k in zip(qs, ks))
        return {"bytes": 16 * (T + case["pad"]) + 12 * n + 8 * new + 4 * used, "flops": 0}
    elt, H, KVH, D = DTYPES[case["dtype"]].itemsize, case["H"], case["KVH"], case["D"]
    nbytes = 2 * sum(ks) * KVH * D * elt + 2 * T * H * D * elt + 4 * T * H + 8 * n
    if case["kind"] == "chunk":
        nbytes += 4 * sum(_blocks(k, case["BS"]) for k in ks)
    if case["kind"] == "chunk" or case["causal"]:
        pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(qs, ks))
    else:
        pairs = sum(q * k for q, k in zip(qs, ks))
    return {"bytes": nbytes, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    """Row by row and head by head, from softmax(scale q K^T) V. Tables are whole numbers: no
    value in 64 bits."""
    if case["kind"] == "tables":
        return None
    st = prepare(case, seed)
    H, KVH, D = case["H"], case["KVH"], case["D"]
    causal = case["kind"] == "chunk" or case["causal"]
    out = torch.empty(st["T"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(H, st["T"], dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for i, (nq, nk) in enumerate(zip(st["qs"], st["ks"])):
        for g in range(KVH):
            if case["kind"] == "chunk":
                ids = st["bt"][i, :_blocks(nk, case["BS"])].long()
                keys = st["k"][ids, :, g].reshape(-1, D)[:nk].double()
                vals = st["v"][ids, :, g].reshape(-1, D)[:nk].double()
            else:
                keys = st["k"][k0:k0 + nk, g].double()
                vals = st["v"][k0:k0 + nk, g].double()
            for h in range(g * (H // KVH), (g + 1) * (H // KVH)):
                s = (st["q"][q0:q0 + nq, h].double() @ keys.t().contiguous()) / math.sqrt(D)
                if causal:
                    s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu_(nk - nq + 1),
                                   float("-inf"))
                z = torch.logsumexp(s, 1)
                out[q0:q0 + nq, h] = torch.exp(s - z[:, None]) @ vals
                lse[h, q0:q0 + nq] = z
        q0 += nq
        k0 += nk
    return out, lse
