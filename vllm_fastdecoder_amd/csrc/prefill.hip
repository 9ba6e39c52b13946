// Attention of packed query tokens: which kernel a call takes, its workspace,
// and the generic kernel that is right for every layout.
#include "prefill_mm.h"

#include <algorithm>
#include <cmath>

namespace fd {

namespace {

// One wave per (query token, head): any head size up to 512, block size,
// stride and type; nothing here is tuned.
__global__ __launch_bounds__(kWave) void prefill_generic_kernel(PrefillArgs a) {
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
  float m, l, acc[8];  // D <= 512
  scalar_attention(a, i, r, t, h, 0, end, m, l, acc);
  scalar_store(a, t, h, m, l, acc);
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

// ------------------------------------------------------------ divided keys
namespace {

// The parts of a token and head's keys, joined: one wave each, lane l holding
// elements 4 l .. + 3 (D = 256 in one go, smaller heads on fewer lanes).
__global__ __launch_bounds__(256) void prefill_combine_kernel(PrefillMmParams p) {
  const PrefillArgs& a = p.a;
  const int lane = threadIdx.x % kWave;
  const int64_t at = (int64_t)blockIdx.x * (256 / kWave) + threadIdx.x / kWave;
  const int64_t all = (int64_t)a.T * a.H;
  if (at >= all) return;
  const int t = (int)(at / a.H), h = (int)(at % a.H);
  const int i = last_row(a.n, t, [&](int r) { return (int64_t)a.cu_q[r]; });
  const PrefillRow r = prefill_row(a, i);
  if (t < r.q0 || t >= r.q0 + r.nq) return;
  const bool small = (int64_t)r.nq * p.G <= kRowsB && p.plan.rows_b > 0;
  const bool is_b = small || p.plan.tiles_a == 0;
  const int parts = is_b ? p.plan.sb : p.plan.sa;
  if (parts <= 1) return;  // written by its own workgroup
  float m = neg_inf();
  for (int s = lane; s < parts; s += kWave) m = fmaxf(m, p.part_ml[s * all + at].x);
  m = wave_max(m);
  const float base = m == neg_inf() ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d = 4 * lane;
  for (int s = 0; s < parts; ++s) {
    const float2 ml = p.part_ml[s * all + at];
    if (ml.y == 0.f) continue;  // no key of this part is seen: nothing was stored
    const float w = fast_exp2(ml.x - base);
    l += w * ml.y;
    if (d < a.D) {
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + (s * all + at) * a.D + d);
      acc.x += w * x.x;
      acc.y += w * x.y;
      acc.z += w * x.z;
      acc.w += w * x.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane == 0)
    a.lse[(int64_t)h * a.lse_sh + t] = l == 0.f ? neg_inf() : (base + fast_log2(l)) * kLn2;
  if (d >= a.D) return;
  const int64_t o = (int64_t)t * a.out_st + (int64_t)h * a.out_sh + d;
  const float y[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(a.out, o + e, a.out_dt, y[e]);
}

int device_cu_count() {
  static thread_local int dev = -1, cus = 0;
  int cur = 0;
  if (hipGetDevice(&cur) != hipSuccess) {
    (void)hipGetLastError();
    return 256;
  }
  if (cur != dev) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, cur) != hipSuccess || n <= 0) {
      (void)hipGetLastError();
      n = 256;
    }
    dev = cur;
    cus = n;
  }
  return cus;
}

bool mm_head_size(int D) { return (D % 16 == 0 && D >= 32 && D <= 128) || D == 256; }

}  // namespace

int launch_prefill_combine(const PrefillMmParams& p, hipStream_t s) {
  const int64_t waves = (int64_t)p.a.T * p.a.H;
  hipLaunchKernelGGL(prefill_combine_kernel, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FD_OK : hip_error(e, "prefill_combine_kernel launch");
}

PrefillPlan plan_prefill_mm(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D, int32_t max_q,
                            int64_t max_k) {
  PrefillPlan pl{};
  const int G = H / KVH;
  const int64_t rows = (int64_t)T * G;
  const int64_t longest = std::min<int64_t>(max_q, T) * G;
  if (longest <= kRowsB) {
    pl.rows_b = n;
  } else if (n == 1) {
    pl.tiles_a = (int32_t)((rows + kRowsA - 1) / kRowsA);
  } else {
    // a row among them may be of any size
    pl.rows_b = n;
    pl.tiles_a = (int32_t)(rows / kRowsA + std::min<int64_t>(n, rows / (kRowsB + 1)));
  }
  // Keys are divided where there are fewer tasks than the CUs hold at once
  // (two workgroups each).
  const int64_t slots = 2LL * device_cu_count();
  const int64_t tasks = ((int64_t)pl.tiles_a + pl.rows_b) * KVH;
  const int64_t steps = (max_k + 63) / 64;
  const int64_t parts = std::max<int64_t>(1, std::min(slots / std::max<int64_t>(tasks, 1), steps / 4));
  pl.sa = pl.tiles_a > 0 ? (int32_t)parts : 1;
  pl.sb = pl.rows_b > 0 ? (int32_t)parts : 1;
  if (parts > 1) pl.workspace = (size_t)parts * T * H * (D * sizeof(float) + sizeof(float2));
  return pl;
}

size_t prefill_workspace_bytes(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D,
                               int32_t max_q, int64_t max_k, int32_t dt) {
  if (!mm_head_size(D)) return 0;
  return plan_prefill_mm(n, T, H, KVH, D, max_q, max_k).workspace;
}

int launch_prefill(const PrefillArgs& a, size_t workspace_bytes, hipStream_t s) {
  (void)workspace_bytes;
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int unit = a.dt == FD_F32 ? 4 : 8;  // elements of 16 bytes
  auto strides = [&](int64_t x, int64_t y) {
    return x >= 0 && y >= 0 && x % unit == 0 && y % unit == 0;
  };
  const bool fast = mm_head_size(a.D) && aligned(a.q) && aligned(a.k) &&
                    aligned(a.v) && aligned(a.out) && strides(a.q_st, a.q_sh) &&
                    strides(a.out_st, a.out_sh) && strides(a.k_st, a.k_sh) &&
                    strides(a.v_st, a.v_sh) && strides(a.k_sb, a.v_sb) &&
                    (int64_t)a.max_q * (a.H / a.KVH) < (1 << 30) && a.max_k < INT32_MAX - 1024;
  if (!fast) return launch_prefill_generic(a, s);
  PrefillMmParams p{};
  p.a = a;
  if (a.bt == nullptr) {  // packed keys: blocks of one
    p.a.k_sb = a.k_st;
    p.a.v_sb = a.v_st;
  }
  p.plan = plan_prefill_mm(a.n, a.T, a.H, a.KVH, a.D, a.max_q, a.max_k);
  p.G = a.H / a.KVH;
  // (a scale of 0 makes all scores alike, which a scale too small to show does
  // too; its product with -inf, a masked score, is still -inf)
  const float scale = a.scale * kLog2e;
  p.q_flip = scale >= 0.f ? 0u : a.dt == FD_F32 ? 0x80000000u : 0x80008000u;
  p.scale_log2 = scale == 0.f ? 0x1p-100f : std::fabs(scale);
  int sh = 0;
  while ((1ll << sh) < a.BS) ++sh;
  p.bs_shift = 31 + sh;
  p.bs_magic = (uint32_t)(((1ull << (31 + sh)) + a.BS - 1) / a.BS);
  if (p.plan.workspace > 0) {
    const int parts = std::max(p.plan.sa, p.plan.sb);
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)parts * a.T * a.H * a.D);
  }
  const int64_t tasks =
      ((int64_t)p.plan.tiles_a * p.plan.sa + (int64_t)p.plan.rows_b * p.plan.sb) * a.KVH;
  if (tasks > INT32_MAX) return set_error(FD_ERR_UNSUPPORTED, "prefill: too many tasks");
  const int rc = a.dt == FD_F16    ? launch_prefill_mm_f16(p, s)
                 : a.dt == FD_BF16 ? launch_prefill_mm_bf16(p, s)
                                   : launch_prefill_mm_f32(p, s);
  if (rc != FD_OK || (p.plan.sa <= 1 && p.plan.sb <= 1)) return rc;
  return launch_prefill_combine(p, s);
}

}  // namespace fd
