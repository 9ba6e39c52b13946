// Block tables, slot mapping, positions and sequence lengths of a step, from
// its requests' lengths (fd_build_tables): the arrays that the cache write,
// the tier planner and the attention calls take, without a host in between.
//
// Row r's new blocks come from the free list at taken + sum_{s < r} need_s.
// A workgroup takes kThreads rows (their table entries and lengths) or
// kThreads tokens (their slots); each finds the sum it needs by adding up the
// needs of the rows ahead of it. That is 12 n bytes from L2 per workgroup at
// most, where a scan by itself would be a launch (or a wait between
// workgroups) of its own: a step's tables are a few dependent memory trips
// either way, never bound by bytes. Workgroups never read what another one
// writes: a token whose block is new takes its id from the free list, as its
// row's table entry does.
#include "fd_common.h"

namespace fd {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct Row {
  int q0, q1, ctx, held, need;
  bool ok;  // its lengths make sense and its table is wide enough
};

__device__ __forceinline__ Row load_row(const BuildTablesArgs& a, int r) {
  Row x;
  x.q0 = a.qsl[r];
  x.q1 = a.qsl[r + 1];
  x.ctx = a.ctx[r];
  const int64_t len = (int64_t)x.ctx + x.q1 - x.q0;
  x.ok = x.q0 >= 0 && x.q0 <= x.q1 && x.q1 <= a.T && x.ctx >= 0 &&
         len <= (int64_t)a.bt_width * a.BS && len <= INT32_MAX;
  x.held = x.ok ? (int)(((int64_t)x.ctx + a.BS - 1) / a.BS) : 0;
  x.need = x.ok && a.free_blocks != nullptr ? (int)((len + a.BS - 1) / a.BS) - x.held : 0;
  return x;
}

struct Shared {
  int64_t wave_total[kWaves];
  int start[kThreads];      // a chunk of rows: query_start_loc,
  int64_t first[kThreads];  // needs of the rows ahead
};

// Sum over the workgroup.
__device__ __forceinline__ int64_t block_sum(int64_t x, Shared& sh) {
  for (int m = kWave / 2; m >= 1; m >>= 1) x += __shfl_xor(x, m, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.wave_total[threadIdx.x / kWave] = x;
  __syncthreads();
  int64_t s = 0;
  for (int w = 0; w < kWaves; ++w) s += sh.wave_total[w];
  return s;
}

// Sum over the threads before this one; *all: over the workgroup.
__device__ __forceinline__ int64_t block_prefix(int64_t x, Shared& sh, int64_t* all) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int64_t in = x;
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t o = __shfl_up(in, d, kWave);
    if (lane >= d) in += o;
  }
  __syncthreads();
  if (lane == kWave - 1) sh.wave_total[wave] = in;
  __syncthreads();
  int64_t ahead = 0, sum = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) ahead += sh.wave_total[w];
    sum += sh.wave_total[w];
  }
  *all = sum;
  return ahead + in - x;
}

// Blocks that rows [0, to) need.
__device__ __forceinline__ int64_t needs_before(const BuildTablesArgs& a, int to, Shared& sh) {
  if (a.free_blocks == nullptr) return 0;
  int64_t s = 0;
  for (int r = threadIdx.x; r < to; r += kThreads) s += load_row(a, r).need;
  return block_sum(s, sh);
}

__device__ __forceinline__ void row_group(const BuildTablesArgs& a, int64_t taken, int r0,
                                          Shared& sh) {
  const int tid = threadIdx.x;
  const int r = r0 + tid;
  Row x{0, 0, 0, 0, 0, true};
  if (r < a.n) x = load_row(a, r);
  const int64_t base = taken + needs_before(a, r0, sh);
  int64_t all;
  const int64_t first = base + block_prefix(x.need, sh, &all);
  // (taken < 0: not a place in the list)
  const bool fits = x.need == 0 || (taken >= 0 && first + x.need <= a.num_free);
  if (r < a.n) {
    a.seq_lens[r] = x.ctx + (x.q1 - x.q0);
    if (x.ok && fits)
      for (int k = 0; k < x.need; ++k)
        a.bt[(int64_t)r * a.bt_stride + x.held + k] = a.free_blocks[first + k];
    if ((!x.ok || !fits) && a.error_count != nullptr) atomicAdd(a.error_count, 1);
  }
  // blocks taken in all: the rows that fit are those ahead of the first that
  // does not (among rows that need any), so the count ends in one group: the
  // one that holds that row, or the last
  if (a.free_blocks != nullptr) {
    const int64_t got = block_sum(fits ? x.need : 0, sh);
    const bool cut = base <= a.num_free && base + all > a.num_free;
    const bool last = r0 + kThreads >= a.n && base + all <= a.num_free;
    if (tid == 0 && taken >= 0 && (cut || last)) *a.taken_out = (int32_t)(base + got);
    if (tid == 0 && (taken < 0 || taken > a.num_free) && r0 == 0) *a.taken_out = (int32_t)taken;
  }
}

__device__ __forceinline__ void token_group(const BuildTablesArgs& a, int64_t taken, int t0,
                                            Shared& sh) {
  const int tid = threadIdx.x;
  const int t = t0 + tid;
  const int t_last = min(a.T, t0 + kThreads) - 1;
  // the last row that starts at or before the group's first token
  int64_t starts = 0;
  for (int r = tid; r < a.n; r += kThreads) starts += a.qsl[r] <= t0 ? 1 : 0;
  const int ra = max(0, (int)block_sum(starts, sh) - 1);
  int64_t ahead = taken + needs_before(a, ra, sh);
  int row = -1;  // of this thread's token
  int64_t first = 0;
  for (int c = ra; c < a.n; c += kThreads) {
    const int rows = min(kThreads, a.n - c);
    const int need = tid < rows ? load_row(a, c + tid).need : 0;
    int64_t all;
    const int64_t mine = ahead + block_prefix(need, sh, &all);
    __syncthreads();
    sh.start[tid] = tid < rows ? a.qsl[c + tid] : INT32_MAX;
    sh.first[tid] = mine;
    __syncthreads();
    if (sh.start[0] <= t) {  // the chunk's last row that starts at or before t
      int lo = 0, hi = rows;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sh.start[mid] <= t)
          lo = mid;
        else
          hi = mid;
      }
      row = c + lo;
      first = sh.first[lo];
    }
    ahead += all;
    if (sh.start[rows - 1] > t_last) break;  // (the same for every thread)
  }
  if (t >= a.T) return;
  int64_t slot = -1, pos = 0;
  if (row >= 0) {
    const Row x = load_row(a, row);
    if (t >= x.q0 && t < x.q1) {
      pos = (int64_t)x.ctx + t - x.q0;
      const bool fits = x.need == 0 || (taken >= 0 && first + x.need <= a.num_free);
      if (x.ok && fits) {
        const int b = (int)(pos / a.BS);
        const int64_t id = b >= x.held && a.free_blocks != nullptr
                               ? a.free_blocks[first + (b - x.held)]
                               : a.bt[(int64_t)row * a.bt_stride + b];
        if (id >= 0 && id < a.num_blocks)
          slot = id * a.BS + pos % a.BS;
        else if (a.error_count != nullptr)
          atomicAdd(a.error_count, 1);
      }
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

__global__ __launch_bounds__(kThreads) void build_tables_kernel(BuildTablesArgs a,
                                                                int row_groups) {
  __shared__ Shared sh;
  const int64_t taken = a.free_blocks != nullptr ? *a.taken_in : 0;
  const int b = (int)blockIdx.x;
  if (b < row_groups)
    row_group(a, taken, b * kThreads, sh);
  else
    token_group(a, taken, (b - row_groups) * kThreads, sh);
}

}  // namespace

int launch_build_tables(const BuildTablesArgs& a, hipStream_t s) {
  int row_groups = (int)(((int64_t)a.n + kThreads - 1) / kThreads);
  if (row_groups == 0 && a.free_blocks != nullptr) row_groups = 1;  // writes taken_out
  const int64_t groups = row_groups + ((int64_t)a.T + kThreads - 1) / kThreads;
  if (groups == 0) return FD_OK;
  hipLaunchKernelGGL(build_tables_kernel, dim3((unsigned)groups), dim3(kThreads), 0, s, a,
                     row_groups);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FD_OK : hip_error(e, "build_tables_kernel launch");
}

}  // namespace fd
