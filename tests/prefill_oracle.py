"""Attention of packed query tokens in 64 bits on the CPU, with the bounds that
its results may be off by, and the inputs of the tests that use it.

Bounds (u = half a step of the type, u32 = 2^-24), for a token with weights
w_k over the keys it sees, scores s_k = scale q . k:
  score    D products and their sum, in any order and with a few roundings per
           step of a matrix instruction: ds = 4 (D + 8) u32 scale max_k sum |q||k|,
           and the scaling and the hardware exp2 and log2 (2^-22 relative and
           2^-23 of the exponent's own size): de = 2^-21 (4 + max_k |s_k|);
  weight   relative error 2 (ds + de) (its own and the sum's), plus u of a
           weight held in 16 bits, plus (L + 8) u32 of the sum over L keys and
           as much of the products' sum;
  out      that times A = sum_k w_k |v_k|, and u |out| of the last rounding
           (+ 2^-24 for results of fp16's smallest sizes, and the same for
           weights there, which leave 2^-24 A);
  lse      ds + de + (L + 8) u32, and 2^-22 |lse| of its own rounding.
"""

from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def visible(nq: int, nk: int, causal: bool) -> torch.Tensor:
    """[nq, nk]: whether token j sees key k."""
    if not causal:
        return torch.ones(nq, nk, dtype=torch.bool)
    return torch.arange(nk)[None, :] <= torch.arange(nq)[:, None] + (nk - nq)


def attend(q, k, v, scale, causal, out_dtype):
    """q [nq, H, D], k / v [nk, KVH, D] on the CPU -> out, lse [nq, H(, D)] in 64 bits and the
    bounds of both. Keys that a token does not see do not enter, whatever they hold."""
    nq, H, D = q.shape
    nk, KVH, _ = k.shape
    see = visible(nq, nk, causal)
    out = torch.zeros(nq, H, D, dtype=torch.float64)
    lse = torch.full((nq, H), -math.inf, dtype=torch.float64)
    tol_o = torch.zeros_like(out)
    tol_l = torch.zeros_like(lse)
    if nk == 0 or nq == 0:
        return out, lse, tol_o, tol_l
    u_w = U[q.dtype] if q.dtype != torch.float32 else 0.0
    for h in range(H):
        g = h // (H // KVH)
        qq, kk, vv = q[:, h].double(), k[:, g].double(), v[:, g].double()
        s = (qq @ kk.t()) * scale
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        big = torch.where(see, qq.abs() @ kk.abs().t(), torch.zeros_like(s)).amax(1) * abs(scale)
        some = see.any(1)
        m = torch.where(some, s.amax(1), torch.zeros(nq, dtype=torch.float64))
        p = torch.exp(s - m[:, None])
        l = p.sum(1)
        w = torch.where(see, p / torch.where(some, l, torch.ones_like(l))[:, None],
                        torch.zeros_like(p))
        # (0 times a value that is not finite must not enter)
        vz = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
        o, a = w @ vz, w @ vz.abs()
        hit = w.gt(0).double()
        for val in (math.inf, -math.inf):
            n = hit @ (vv == val).double()
            o = torch.where(n > 0, o + val, o)
        o = torch.where(hit @ torch.isnan(vv).double() > 0, torch.full_like(o, math.nan), o)
        out[:, h] = torch.where(some[:, None], o, torch.zeros_like(o))
        lse[:, h] = torch.where(some, m + torch.log(torch.where(some, l, torch.ones_like(l))), lse[:, h])
        L = see.sum(1).double()
        ds = 4 * (D + 8) * 2.0 ** -24 * big
        smax = torch.where(see, s.abs(), torch.zeros_like(s)).amax(1)
        de = 2.0 ** -21 * (4 + smax)
        rel = 2 * (ds + de) + u_w + 2 * (L + 8) * 2.0 ** -24
        tol_o[:, h] = rel[:, None] * a + U[out_dtype] * o.abs() + 2.0 ** -24 * (1 + a)
        tol_l[:, h] = ds + de + (L + 8) * 2.0 ** -24 + 2.0 ** -22 * torch.where(
            some, lse[:, h].abs(), torch.zeros(nq, dtype=torch.float64))
    return out, lse, tol_o, tol_l


def check(got_o, got_l, ref, what=""):
    """got_o [nq, H, D], got_l [H, nq] against attend()'s answer."""
    o, lse, tol_o, tol_l = ref
    got_o, got_l = got_o.double().cpu(), got_l.t().double().cpu()
    assert torch.equal(torch.isnan(got_o), torch.isnan(o)), f"{what}: NaN elsewhere"
    inf = torch.isinf(o)
    assert torch.equal(got_o[inf], o[inf]), f"{what}: infinities"
    fin = torch.isfinite(o)
    off = ((got_o - o).abs() - tol_o)[fin]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: out off by {float(off.max()):.3g} more than its bound"
    empty = torch.isneginf(lse)
    assert torch.equal(torch.isneginf(got_l), empty), f"{what}: lse of tokens without keys"
    off = ((got_l - lse).abs() - tol_l)[~empty]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: lse off by {float(off.max()):.3g} more than its bound"


def starts(lens) -> torch.Tensor:
    return torch.tensor([0] + list(lens), dtype=torch.int32).cumsum(0).to(torch.int32)


class Paged:
    """Rows of qs new tokens and ks tokens in all over a paged cache whose unused entries hold
    NaN: blocks that no row has, and the last blocks' tails."""

    def __init__(self, qs, ks, H, KVH, D, dtype, BS=16, seed=0, extra_cols=0, pad=0, amp=1.0):
        g = torch.Generator().manual_seed(seed)
        self.qs, self.ks, self.BS, self.D = list(qs), list(ks), BS, D
        n = len(self.qs)
        counts = [-(-k // BS) for k in self.ks]
        self.B = sum(counts) + 3
        ids = torch.randperm(self.B, generator=g)
        W = max(max(counts, default=0), 1) + extra_cols
        self.bt = torch.full((n, W), -7, dtype=torch.int32)
        kv = torch.full((self.B, BS, KVH, 2 * D), math.nan, dtype=dtype)
        self.k, self.v = [], []
        pos = 0
        for i, (c, nk) in enumerate(zip(counts, self.ks)):
            mine = ids[pos:pos + c]
            pos += c
            self.bt[i, :c] = mine.int()
            k = (torch.randn(nk, KVH, D, generator=g) * amp).to(dtype)
            v = torch.randn(nk, KVH, D, generator=g).to(dtype)
            self.k.append(k)
            self.v.append(v)
            for b in range(c):
                lo, hi = b * BS, min((b + 1) * BS, nk)
                kv[mine[b], : hi - lo, :, :D] = k[lo:hi]
                kv[mine[b], : hi - lo, :, D:] = v[lo:hi]
        self.kv = kv
        self.T = sum(self.qs) + pad
        self.q = torch.randn(self.T, H, D, generator=g).to(dtype)
        self.cu = starts(self.qs)
        self.lens = torch.tensor(self.ks, dtype=torch.int32)

    def refs(self, scale, causal, out_dtype):
        q0 = 0
        for nq, k, v in zip(self.qs, self.k, self.v):
            yield q0, nq, attend(self.q[q0:q0 + nq], k, v, scale, causal, out_dtype)
            q0 += nq
