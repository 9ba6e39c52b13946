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

// ------------------------------------------------------------ the plan
namespace {

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

// Keys of a step of the matrix-core kernel (PfShape).
int64_t step_keys(int D, int dt) { return dtype_size(dt) * D <= 256 ? 64 : 32; }

// Runs that a part's table has room for: with V's own beside K's, two stages of
// K and V fit the LDS too.
int64_t table_room(int D, int dt) {
  const int64_t stage = 2 * step_keys(D, dt) * D * (int64_t)dtype_size(dt);
  return std::min<int64_t>(kTableRoom, (kPrefillLds - 2 * stage) / 16);
}

// Keys that lie one after another for certain, in a block of BS or (BS = 0)
// packed, up to kMostRun, as a power of two.
int run_shift(int BS) {
  int s = 0;
  while ((1 << s) < kMostRun && (BS == 0 || BS % (2 << s) == 0)) ++s;
  return s;
}

int32_t prefill_counter_stride(int64_t pairs) {
  return pairs <= kMaxPrefillCounters ? counter_stride(pairs) : 1;
}

// Into how many parts an A tile's keys are cut. A model of the time, in steps:
// each part adds a start and an end, and parts are joined. Alike tiles (one
// row) run in whole rounds; of different rows' tiles about half the work that
// the longest row makes of them is there (the lengths are known on the GPU
// alone), and three quarters of one part are waited for at the end. The start
// and the join, from kernel traces: 12 to 18 and 10 us, a step 2.5 us (16-bit,
// two workgroups on a CU; D = 256: 1.5, alone; fp32: 9). Measured, undivided /
// as this divides / at its best: 4 chunks of 389 to 640 tokens over at most
// 2048 keys, bf16 97 / 94 / 88 us; 3 of 200 to 700 over up to 4000, D = 256,
// 121 / 101 / 101; 3 of 100 to 300 over up to 1500, fp32, 188 / 151 / 151.
int64_t tile_parts(int n, int64_t tasks, int64_t steps, int64_t slots, int D, int dt) {
  const double start = dt == FD_F32 ? 2 : D > 128 ? 10 : 7;
  const double join = dt == FD_F32 ? 2 : D > 128 ? 12 : 6;
  double least = 0, cost[kMostTileParts + 1];
  const int64_t most = std::min<int64_t>(kMostTileParts, steps);
  for (int64_t parts = 1; parts <= most; ++parts) {
    const double part = (double)((steps + parts - 1) / parts) + start;
    double& c = cost[parts];
    if (n == 1) {
      c = (double)((tasks * parts + slots - 1) / slots) * part;
    } else {
      const double work = 0.5 * (double)tasks * ((double)steps + (double)parts * start) / (double)slots;
      c = std::max(part, work + 0.75 * part);
    }
    if (parts > 1) c += join;
    least = parts == 1 ? c : std::min(least, c);
  }
  int64_t parts = 1;
  while (cost[parts] > least * (1 + 1.0 / 32)) ++parts;  // the fewest of about as good
  return parts;
}

bool mm_head_size(int D) { return (D % 16 == 0 && D >= 32 && D <= 128) || D == 256; }

}  // namespace

PrefillPlan plan_prefill_mm(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D, int32_t max_q,
                            int64_t max_k, int32_t BS, int32_t dt) {
  PrefillPlan pl{};
  const int G = H / KVH;
  const int64_t rows = (int64_t)T * G;
  const int64_t longest = std::min<int64_t>(max_q, T) * G;
  const int64_t keys = step_keys(D, dt);
  const int64_t steps = std::max<int64_t>(1, (max_k + keys - 1) / keys);
  const int64_t cus = device_cu_count();
  // Eight waves where their tiles alone keep every CU busy for long: they
  // read K and V half as often (bf16, 32 / 8 heads of 128, 4096 tokens over
  // 28000 keys: 1874 us, with four waves 2326). Two workgroups of four share a
  // CU, and one computes while the other starts or ends: better for short
  // ones (16 fresh prompts of up to 512 tokens, 32 heads of 128: 52 us, with
  // eight waves 62; four chunks of 389 to 640 tokens over at most 2048 keys:
  // 97 and 115).
  const int64_t wide = (rows + 255) / 256 * KVH;
  pl.waves = D <= 128 && longest > kRowsB && steps >= 64 && wide >= (n == 1 ? cus : 2 * cus) ? 8 : 4;
  const int rows_a = 32 * pl.waves;
  if (longest <= kRowsB) {
    pl.rows_b = n;
  } else if (n == 1) {
    pl.tiles_a = (int32_t)((rows + rows_a - 1) / rows_a);
  } else {
    // a row among them may be of any size
    pl.rows_b = n;
    pl.tiles_a = (int32_t)(rows / rows_a + std::min<int64_t>(n, rows / (kRowsB + 1)));
  }
  const int64_t tasks = ((int64_t)pl.tiles_a + pl.rows_b) * KVH;
  const int64_t slots = D > 128 || pl.waves == 8 ? cus : 2 * cus;  // workgroups at once
  pl.per_a = pl.per_b = (int32_t)steps;
  if (tasks <= kMaxPrefillCounters) {
    const int64_t parts_a = tile_parts(n, tasks, steps, slots, D, dt);
    pl.per_a = (int32_t)((steps + parts_a - 1) / parts_a);
    // A row's few tokens, which its K and V's way from memory bounds: as many
    // parts as run at once, of two steps at least (one row of 5 tokens, 900
    // keys, 8 kv heads: 14.9 us, with parts of 1 step 16.2, of 4 17.1,
    // undivided 26). Of many rows most are shorter than the longest: some more
    // (48 rows of 2 to 9 tokens, up to 3100 keys, 4 kv heads: parts of 16
    // steps 42 us, of 24 44, of 12 55, undivided 57).
    const int64_t most = n == 1 ? slots : slots + slots / 4;
    const int64_t parts = std::max<int64_t>(1, most / tasks);
    pl.per_b = (int32_t)std::min(steps, std::max<int64_t>(2, (steps + parts - 1) / parts));
  }
  // a part's keys as far as their table has room
  const int64_t most = ((int64_t)(table_room(D, dt) - 2) << run_shift(BS)) / keys;
  pl.per_a = (int32_t)std::min<int64_t>(pl.per_a, most);
  pl.per_b = (int32_t)std::min<int64_t>(pl.per_b, most);
  pl.parts_a = pl.tiles_a > 0 ? (int32_t)((steps + pl.per_a - 1) / pl.per_a) : 1;
  pl.parts_b = pl.rows_b > 0 ? (int32_t)((steps + pl.per_b - 1) / pl.per_b) : 1;
  const int64_t parts = std::max(pl.parts_a, pl.parts_b);
  if (parts > 1) {
    const size_t row = D * sizeof(float) + sizeof(float2);
    pl.partial_bytes = ((size_t)parts * T * H * row + 255) / 256 * 256;
    pl.counter_bytes = (size_t)tasks * prefill_counter_stride(tasks) * sizeof(uint64_t);
  }
  return pl;
}

size_t prefill_workspace_bytes(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D,
                               int32_t max_q, int64_t max_k, int32_t BS, int32_t dt) {
  if (!mm_head_size(D)) return 0;
  const PrefillPlan pl = plan_prefill_mm(n, T, H, KVH, D, max_q, max_k, BS, dt);
  return pl.partial_bytes + pl.counter_bytes;
}

int launch_prefill(const PrefillArgs& a, hipStream_t s) {
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int unit = a.dt == FD_F32 ? 4 : 8;  // elements of 16 bytes
  auto strides = [&](int64_t x, int64_t y) {
    return x >= 0 && y >= 0 && x % unit == 0 && y % unit == 0;
  };
  const bool fast = mm_head_size(a.D) && aligned(a.q) && aligned(a.k) &&
                    aligned(a.v) && aligned(a.out) && strides(a.q_st, a.q_sh) &&
                    strides(a.out_st, a.out_sh) && strides(a.k_st, a.k_sh) &&
                    strides(a.v_st, a.v_sh) && strides(a.k_sb, a.v_sb) &&
                    (int64_t)a.T * (a.H / a.KVH) < (1 << 30) && a.max_k < INT32_MAX - 1024 &&
                    std::max(a.k_st, a.v_st) < (1 << 30);
  if (!fast) return launch_prefill_generic(a, s);
  PrefillMmParams p{};
  p.a = a;
  if (a.bt == nullptr) {  // packed keys: blocks of one
    p.a.k_sb = a.k_st;
    p.a.v_sb = a.v_st;
  }
  p.plan = plan_prefill_mm(a.n, a.T, a.H, a.KVH, a.D, a.max_q, a.max_k,
                           a.bt != nullptr ? a.BS : 0, a.dt);
  const PrefillPlan& pl = p.plan;
  p.G = a.H / a.KVH;
  // (a scale of 0 makes all scores alike, which a scale too small to show does
  // too; its product with -inf, a masked score, is still -inf)
  const float scale = a.scale * kLog2e;
  p.q_flip = scale >= 0.f ? 0u : a.dt == FD_F32 ? 0x80000000u : 0x80008000u;
  p.scale_log2 = scale == 0.f ? 0x1p-100f : std::fabs(scale);
  const int64_t keys = step_keys(a.D, a.dt);
  p.run_shift = run_shift(a.bt != nullptr ? a.BS : 0);
  const int64_t per = std::max(pl.tiles_a > 0 ? pl.per_a : 0, pl.rows_b > 0 ? pl.per_b : 0);
  p.table_room = (int32_t)(((per * keys) >> p.run_shift) + 2);
  p.grid = ((int64_t)pl.tiles_a * pl.parts_a + (int64_t)pl.rows_b * pl.parts_b) * a.KVH;
  if (p.grid > INT32_MAX) return set_error(FD_ERR_UNSUPPORTED, "prefill: too many tasks");
  p.alone = p.grid <= device_cu_count();
  if (pl.partial_bytes > 0) {
    const int parts = std::max(pl.parts_a, pl.parts_b);
    const int64_t pairs = ((int64_t)pl.tiles_a + pl.rows_b) * a.KVH;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (size_t)parts * a.T * a.H * a.D);
    p.counters = pairs <= kMaxPrefillCounters ? a.counters : nullptr;
    p.counter_stride = prefill_counter_stride(pairs);
    p.launch = next_launch() << kLaunchBits;
    if (p.counters == nullptr) {
      p.counters = reinterpret_cast<uint64_t*>(static_cast<char*>(a.workspace) + pl.partial_bytes);
      const int rc = launch_clear_counters(p.counters, (int32_t)pairs, p.counter_stride, s);
      if (rc != FD_OK) return rc;
    }
  }
  return a.dt == FD_F16    ? launch_prefill_mm_f16(p, s)
         : a.dt == FD_BF16 ? launch_prefill_mm_bf16(p, s)
                           : launch_prefill_mm_f32(p, s);
}

}  // namespace fd
