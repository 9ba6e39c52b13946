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

int launch_prefill_generic(const PrefillArgs& a, hipStream_t s);

}  // namespace fd
