// Attention of packed query tokens: which kernel a call takes, its workspace,
// and the generic kernel that is right for every layout.
#include "prefill.h"

namespace fd {

namespace {

// One wave per (query token, head), lane l holding elements l + 64 k: any head
// size up to 512, block size, stride and type. Keys one after another with a
// running maximum and sum; nothing here is tuned.
__global__ __launch_bounds__(kWave) void prefill_generic_kernel(PrefillArgs a) {
  constexpr int kMaxPerLane = 8;  // D <= 512
  const int lane = threadIdx.x;
  const int h = blockIdx.x % a.H;
  const int t = blockIdx.x / a.H;
  const int i = last_row(a.n, t, [&](int r) { return (int64_t)a.cu_q[r]; });
  const PrefillRow r = prefill_row(a, i);
  const int j = t - r.q0;
  if (j < 0 || j >= r.nq) return;  // in no row: left as it is
  bool bad = r.bad;
  if (a.bt != nullptr) {  // every block of the row, seen by this token or not
    const int nb = (int)(((int64_t)r.nk + a.BS - 1) / a.BS);
    for (int b = lane; b < nb; b += kWave) {
      const int64_t id = a.bt[(int64_t)i * a.bt_stride + b];
      bad |= id < 0 || id >= a.num_blocks;
    }
    bad = __ballot(bad) != 0;
  }
  const int64_t obase = (int64_t)t * a.out_st + (int64_t)h * a.out_sh;
  const int end = bad ? 0 : last_key(a, r, j) + 1;
  if (end <= 0) {
    for (int d = lane; d < a.D; d += kWave) store_elem(a.out, obase + d, a.out_dt, bad ? qnan() : 0.f);
    if (lane == 0) a.lse[(int64_t)h * a.lse_sh + t] = bad ? qnan() : neg_inf();
    return;
  }
  const int kh = h / (a.H / a.KVH);
  float qv[kMaxPerLane], acc[kMaxPerLane];
  const int64_t qbase = (int64_t)t * a.q_st + (int64_t)h * a.q_sh;
#pragma unroll
  for (int x = 0; x < kMaxPerLane; ++x) {
    const int d = lane + x * kWave;
    qv[x] = d < a.D ? load_elem(a.q, qbase + d, a.dt) : 0.f;
    acc[x] = 0.f;
  }
  float m = neg_inf(), l = 0.f;
  for (int key = 0; key < end; ++key) {
    int64_t kb, vb;
    if (a.bt != nullptr) {
      const int64_t id = a.bt[(int64_t)i * a.bt_stride + key / a.BS];
      kb = id * a.k_sb + (int64_t)(key % a.BS) * a.k_st;
      vb = id * a.v_sb + (int64_t)(key % a.BS) * a.v_st;
    } else {
      kb = (int64_t)(r.k0 + key) * a.k_st;
      vb = (int64_t)(r.k0 + key) * a.v_st;
    }
    kb += (int64_t)kh * a.k_sh;
    vb += (int64_t)kh * a.v_sh;
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < kMaxPerLane; ++x) {
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
    for (int x = 0; x < kMaxPerLane; ++x) {
      const int d = lane + x * kWave;
      if (d < a.D) acc[x] = acc[x] * alpha + p * load_elem(a.v, vb + d, a.dt);
    }
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int x = 0; x < kMaxPerLane; ++x) {
    const int d = lane + x * kWave;
    if (d < a.D) store_elem(a.out, obase + d, a.out_dt, acc[x] * inv);
  }
  if (lane == 0) a.lse[(int64_t)h * a.lse_sh + t] = l == 0.f ? neg_inf() : m + __logf(l);
}

}  // namespace

int launch_prefill_generic(const PrefillArgs& a, hipStream_t s) {
  if ((int64_t)a.T * a.H > INT32_MAX)
    return set_error(FD_ERR_UNSUPPORTED, "prefill: too many (token, head) pairs");
  hipLaunchKernelGGL(prefill_generic_kernel, dim3((unsigned)((int64_t)a.T * a.H)), dim3(kWave), 0,
                     s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FD_OK : hip_error(e, "prefill_generic_kernel launch");
}

size_t prefill_workspace_bytes(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D,
                               int32_t max_q, int64_t max_k, int32_t dt) {
  return 0;
}

int launch_prefill(const PrefillArgs& a, size_t workspace_bytes, hipStream_t s) {
  return launch_prefill_generic(a, s);
}

}  // namespace fd
