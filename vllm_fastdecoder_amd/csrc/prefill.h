// What the kernels of packed query tokens share (fd_paged_prefill,
// fd_varlen_attention): a row's tokens and keys, checked on the device, and
// the search for the row that a workgroup works on.
#pragma once

#include "fd_common.h"

namespace fd {

// One row: its query tokens [q0, q0 + nq) and its nk keys; packed keys start
// at k0. nq = 0: nothing to write (an empty row, or one whose query tokens do
// not lie in the call's). bad: a range error, the row's results are NaN.
struct PrefillRow {
  int q0, nq, k0, nk;
  bool bad;
};

__device__ __forceinline__ PrefillRow prefill_row(const PrefillArgs& a, int i) {
  PrefillRow r{a.cu_q[i], 0, 0, 0, false};
  const int q1 = a.cu_q[i + 1];
  if (r.q0 < 0 || q1 < r.q0 || q1 > a.T) return r;
  r.nq = q1 - r.q0;
  r.bad = r.nq > a.max_q;
  if (a.bt != nullptr) {
    r.nk = max(a.lens[i], 0);
    r.bad |= r.nk > (int64_t)a.bt_width * a.BS || (r.nk > 0 && a.num_blocks <= 0);
  } else {
    r.k0 = a.cu_k[i];
    const int k1 = a.cu_k[i + 1];
    r.bad |= r.k0 < 0 || k1 < r.k0 || k1 > a.Tk || k1 - r.k0 > a.max_k;
    r.nk = k1 - r.k0;
  }
  if (r.bad) r.nk = 0;
  return r;
}

// The last key that token j of the row sees (-1: none).
__device__ __forceinline__ int last_key(const PrefillArgs& a, const PrefillRow& r, int j) {
  return a.causal ? min(r.nk - 1, r.nk - r.nq + j) : r.nk - 1;
}

// The last row i of n with f(i) <= x, f not decreasing (0 where none); by a
// whole wave, 64 rows a round.
template <typename F>
__device__ __forceinline__ int last_row(int n, int64_t x, F&& f) {
  const int lane = threadIdx.x % kWave;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + kWave - 1) / kWave;
    const int at = lo + lane * step;
    const uint64_t le = __ballot(lane * step < len && f(at) <= x);
    // (rows behind the first that lies past x do not count, should the
    // caller's starts not be in order)
    const int k = le == ~0ull ? kWave : __builtin_ctzll(~le);
    const int next = lo + max(k - 1, 0) * step;
    len = min(step, lo + len - next);
    lo = next;
    if (step == 1) break;
  }
  return lo;
}

// One query token and head over keys [from, to) of its row, one key after
// another with a running maximum and sum, by a wave: lane l holds elements
// l + 64 k of the head. acc is the sum of weights exp(s - m) times V.
template <int kPerLane>
__device__ __forceinline__ void scalar_attention(const PrefillArgs& a, int i, const PrefillRow& r,
                                                 int t, int h, int from, int to, float& m, float& l,
                                                 float (&acc)[kPerLane]) {
  const int lane = threadIdx.x % kWave;
  const int kh = h / (a.H / a.KVH);
  const bool paged = a.bt != nullptr;
  float qv[kPerLane];
  const int64_t qbase = (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
  for (int x = 0; x < kPerLane; ++x) {
    const int d = lane + x * kWave;
    qv[x] = d < a.D ? load_elem(a.q, qbase + d, a.dt) : 0.f;
    acc[x] = 0.f;
  }
  m = neg_inf();
  l = 0.f;
  for (int key = from; key < to; ++key) {
    const int64_t id = paged ? a.bt[(int64_t)i * a.bt_stride + key / a.BS] : r.k0 + key;
    const int64_t in = paged ? key % a.BS : 0;
    const int64_t kb = id * (paged ? a.k_sb : a.k_st) + in * a.k_st + (int64_t)kh * a.k_sh;
    const int64_t vb = id * (paged ? a.v_sb : a.v_st) + in * a.v_st + (int64_t)kh * a.v_sh;
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < kPerLane; ++x) {
      const int d = lane + x * kWave;
      if (d < a.D) s += qv[x] * load_elem(a.k, kb + d, a.dt);
    }
    s = wave_sum(s) * a.scale;
    const float mn = fmaxf(m, s);
    const float base = mn == neg_inf() ? 0.f : mn;  // every score so far -inf
    const float alpha = __expf(m - base);
    const float p = __expf(s - base);
    l = l * alpha + p;
#pragma unroll
    for (int x = 0; x < kPerLane; ++x) {
      const int d = lane + x * kWave;
      if (d < a.D) acc[x] = acc[x] * alpha + p * load_elem(a.v, vb + d, a.dt);
    }
    m = mn;
  }
}

// Its result as out and lse.
template <int kPerLane>
__device__ __forceinline__ void scalar_store(const PrefillArgs& a, int t, int h, float m, float l,
                                             const float (&acc)[kPerLane]) {
  const int lane = threadIdx.x % kWave;
  const int64_t obase = (int64_t)t * a.out_st + (int64_t)h * a.out_sh;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int x = 0; x < kPerLane; ++x) {
    const int d = lane + x * kWave;
    if (d < a.D) store_elem(a.out, obase + d, a.out_dt, acc[x] * inv);
  }
  if (lane == 0) a.lse[(int64_t)h * a.lse_sh + t] = l == 0.f ? neg_inf() : m + __logf(l);
}

int launch_prefill_generic(const PrefillArgs& a, hipStream_t s);

}  // namespace fd
