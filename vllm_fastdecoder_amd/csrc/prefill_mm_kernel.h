// Attention of packed query tokens with both products on the matrix cores,
// instantiated per type by prefill_mm_f16.hip, prefill_mm_bf16.hip and
// prefill_mm_f32.hip.
//
// A workgroup takes a tile of query rows of one kv head and walks a part of the
// tile's keys, 64 a step (32 where a row's D elements pass 256 bytes). Query
// rows are (token, head of the kv head's group) pairs, so grouped-query heads
// share every K and V read and a few tokens of many heads fill a tile as well
// as many tokens of one. Each wave has 32 rows. A tiles: four or eight waves'
// rows, each with all of a step's keys; B tiles: 64 rows of a request with few
// tokens, which the read of K and V bounds: the waves stand 2 rows x 2 parts of
// a step's keys (of eight waves 4 x 2, half of them idle).
//
// Per step and wave, all transposed, so that a lane owns one query row (column
// l % 32 of both products; its half l / 32 of the keys, then of the dims):
//   S^T[key][row] = K Q^T   v_mfma_f32_32x32x16, K from LDS, Q in registers;
//   softmax         a lane's keys in registers, one swap between the halves
//                   for the maximum; a running maximum raised only when a step
//                   passes it by more than kLazyRescale (p <= 2^8), and the
//                   accumulators rescaled then alone;
//   O^T[dim][row] += V^T P^T   P is the B operand as it lies in the S^T
//                   accumulator: lane half h holds keys 4 h .. + 3 and
//                   8 + 4 h .. + 3 of each 16, and V^T's A operand is read in
//                   that order (two ds_read_b64_tr_b16, whose lane mapping is
//                   told in decode_mm.hip), so no lane ever moves a weight.
// fp32 goes the same way with v_mfma_f32_32x32x2: a chunk of 16 bytes is an
// operand of four products (whose two dims are 4 apart, in K and Q alike), and
// the weights are P^T's operand without a conversion.
// P is rounded to the inputs' type (fp16: scaled by 2^7, so that small weights
// stay normal), its sum is taken in fp32 before the rounding; the error it
// adds is of the size of the output's own rounding.
//
// K and V go to LDS by global_load_lds (16 bytes a lane, no registers) in two
// to four stages: a stage is a step's V and the next step's K, as step t's
// weights are computed while the products for step t + 1's scores run, and then
// multiply V; one barrier a step. Where a step's keys lie stands in a table in
// LDS that the workgroup fills first (block ids checked there, once). The
// loads land in order of lanes, so the bank swizzle is in the address that a
// lane reads: LDS slot c of a K row holds chunk c ^ swizzle_k(row), of a V row
// chunk c ^ swizzle_v(row); K is read 16 rows x 16 bytes at a time, V 4 rows x
// 64 bytes.
//
// Keys that no row of a wave sees are skipped, steps that some row sees in
// part are masked (a key against the row's last). What the masked V rows hold
// does not matter as long as it is finite (weight 0); where a result is not
// finite, the workgroup does its part again key by key, each row with the keys
// that it sees.
//
// What bounds it (bf16, 32 / 8 heads of 128): the wave's own issue of
// instructions. A step of a wave is 1024 cycles of matrix instructions beside
// about 210 VALU instructions (32 exponents, sums, fmas for the exponents, 16
// conversions and maxima of three, the loads' addresses) and 52 LDS instructions,
// which overlap only as far as the two waves of a SIMD are in different phases.
// 8 waves, 4096 tokens over 28000 keys: 1815 us, 1.11 PFLOP/s (a large matrix
// product reaches 1.20). The same with every operand read right ahead of its
// product 2331 us; with the weights computed between the two products 2078; with
// scores copied, then turned into exponents as the weights are made (32 VALU
// instructions more) 1900. D = 256: 0.8 PFLOP/s (one wave a SIMD); fp32: 0.130 of
// 0.153.
#pragma once

#include <algorithm>
#include <type_traits>

#include "prefill_mm.h"

namespace fd {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_v __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_ptr;

constexpr float kLazyRescale = 8.f;  // log2 units
constexpr int kReadAhead = 4;        // operands read ahead of their product

template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  static_assert(!std::is_same<T, F32>::value, "16-bit types");
  if constexpr (std::is_same<T, F16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Two fp32 values as a word of two 16-bit ones, rounded to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (std::is_same<T, F16>::value) {
    half2_t h;
    h.x = (_Float16)x;
    h.y = (_Float16)y;
    return __builtin_bit_cast(uint32_t, h);
  } else {
    bf162_t h;
    h.x = (__bf16)x;
    h.y = (__bf16)y;
    return __builtin_bit_cast(uint32_t, h);
  }
}

// 16 bytes per lane from g to LDS at `lds` (the wave's first lane; lane l's
// land 16 l further). As asm: the compiler would wait for it at the next LDS
// read of any kind. It has no register result; whoever reads the bytes waits
// with vmcnt and a barrier. (One instruction between the write of M0 and its
// use.)
__device__ __forceinline__ void load_lds16(const char* g, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(lds), "v"(g)
      : "memory");
}

// Rows of kBytes in LDS: kPeriod rows start at different multiples of the 256
// bytes that all banks serve at once. (fp32 V rows are read 32 floats in a
// row at a time and need none.)
template <int kBytes, bool kF32>
struct Swizzle {
  static constexpr int kPeriod = kBytes % 256 == 0 ? 1 : kBytes % 128 == 0 ? 2 : kBytes % 64 == 0 ? 4 : 8;
  static __device__ __forceinline__ int k(int row) { return (row / kPeriod) & (16 / kPeriod - 1); }
  static __device__ __forceinline__ int v(int row) {
    return !kF32 && kPeriod < 4 ? ((row / kPeriod) & (4 / kPeriod - 1)) << 2 : 0;
  }
};

// NW: waves of a workgroup.
template <typename T, int D, int NW>
struct PfShape {
  static constexpr bool kF32 = std::is_same<T, F32>::value;
  static constexpr int kElt = kF32 ? 4 : 2;
  static constexpr int kThreads = NW * kWave;
  static constexpr int kStepKeys = kElt * D <= 256 ? 64 : 32;  // keys of a step
  static constexpr int kRowBytes = D * kElt;
  static constexpr int kRowsA = 32 * NW;
  static constexpr int kStageBytes = 2 * kStepKeys * kRowBytes;  // K and V of a step
  // waves a SIMD holds: two workgroups of four waves where two stages of both
  // fit the LDS, or one of eight (D = 256: a wave that has a SIMD to itself has
  // twice the registers, which its accumulators need; 224 us for the chunks of
  // the planner's example without, 129 with them)
  static constexpr int kWavesPerSimd = D <= 128 && (NW == 8 || 2 * kStageBytes <= 64 * 1024) ? 2 : 1;
  static constexpr int kPad = 32 * kElt;  // behind the stages: reads past D in the last row
  // the merge of a B tile's two key waves: fp32 accumulators of its rows
  static constexpr int kMergeBytes = kRowsB * ((D + 31) / 32 * 32) * 4;
};

// kCount products, each behind the LDS reads of the operand kAhead products
// further on: read(x) gives product x's operand, use(x, operand) computes it,
// beside(x) is other work that goes on while the product runs, and next(y)
// gives operand y of the products that come after these, whose first kAhead
// are read here. buf: operands in reading order, the first at slot kFirst;
// filled: the first kAhead are there already. In this order by force: left to
// itself the compiler reads each operand right ahead of its product, which then
// waits for it, and keeps the other work apart.
template <int kCount, int kAhead, int kFirst, typename R, typename U, typename B, typename N>
__device__ __forceinline__ void products(u32x4 (&buf)[kAhead], bool filled, R&& read, U&& use,
                                         B&& beside, N&& next) {
  static_assert(kCount >= kAhead, "the products that follow take over the slots");
  if (!filled) {
#pragma unroll
    for (int x = 0; x < kAhead; ++x) buf[(kFirst + x) % kAhead] = read(x);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int x = 0; x < kCount; ++x) {
    u32x4& slot = buf[(kFirst + x) % kAhead];
    use(x, slot);
    slot = x + kAhead < kCount ? read(x + kAhead) : next(x + kAhead - kCount);
    beside(x);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Keeps x's computation where it stands (the compiler is free to move what has
// no effect of its own past a scheduling barrier, and does).
template <typename X>
__device__ __forceinline__ void stay(X& x) {
  asm volatile("" : "+v"(x));
}

// The first lane's value, known to be every lane's.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

template <int NW>
struct PfShared {
  float ml[NW][2][32];
  int last;
};

// A workgroup's task: part `part` (of `parts`, each p.per steps) of the keys of
// rows [row0, row0 + count) of row i's nq * G, for kv head kvh.
struct PfTask {
  int i, row0, count, kvh, part, parts, seen, steps, per;
};

// Partial results are written and read at agent scope (past the XCD's own
// L2), as a tile's parts run on several XCDs.
constexpr int kAgentScope = 16;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t pf_rsrc(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0,
                                           (int)min(bytes, (int64_t)INT32_MAX), 0x00020000);
}

// The partial results of a part of a task's rows: a pair of each row (maximum
// in the log2 domain, sum of weights; a sum of 0: no key, and no sums stored),
// and D sums of each, 32 rows together: four dims of the 32, then the next
// four, so that a wave's accumulators are written and read in whole lines.
struct PfPartial {
  __amdgpu_buffer_rsrc_t o, ml;
  int rows;
  __device__ __forceinline__ PfPartial(const PrefillMmParams& p, const PfTask& task,
                                       const PrefillRow& r, int part) {
    const PrefillArgs& a = p.a;
    const int64_t all = (int64_t)a.T * p.G;
    const int64_t first = ((int64_t)part * a.KVH + task.kvh) * all + (int64_t)r.q0 * p.G + task.row0;
    rows = min(task.count, r.nq * p.G - task.row0);
    o = pf_rsrc(p.part_o + first * a.D, (int64_t)rows * a.D * 4);
    ml = pf_rsrc(p.part_ml + first, (int64_t)rows * 8);
  }
  // byte of dims 4 piece .. + 3 of the task's row x
  __device__ __forceinline__ uint32_t at(int D, int x, int piece) const {
    const int group = x / 32;
    return (group * 32 * D + (piece * min(32, rows - 32 * group) + x % 32) * 4) * 4;
  }
  __device__ __forceinline__ void store_ml(int x, float m, float l) const {
    const uint2_v y = {__float_as_uint(m), __float_as_uint(l)};
    __builtin_amdgcn_raw_buffer_store_b64(y, ml, x * 8, 0, kAgentScope);
  }
  __device__ __forceinline__ void store4(uint32_t at, const float* y) const {
    const u32x4 x = {__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                     __float_as_uint(y[3])};
    __builtin_amdgcn_raw_buffer_store_b128(x, o, at, 0, kAgentScope);
  }
  __device__ __forceinline__ void store1(uint32_t at, float y) const {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y), o, at, 0, kAgentScope);
  }
};

// Four values of a row of out.
template <typename T>
__device__ __forceinline__ void pf_store4(const PrefillArgs& a, int64_t o, const float* y) {
  if (std::is_same<T, F32>::value || a.out_dt == FD_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + o) = make_float4(y[0], y[1], y[2], y[3]);
  } else if constexpr (!std::is_same<T, F32>::value) {
    uint2 u;
    u.x = to_out(T{}, y[0]) | ((uint32_t)to_out(T{}, y[1]) << 16);
    u.y = to_out(T{}, y[2]) | ((uint32_t)to_out(T{}, y[3]) << 16);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) = u;
  }
}

// Waits until at most `stages` later stages of kPerStage loads are under way.
template <int kPerStage>
__device__ __forceinline__ void wait_loads(int stages) {
  static_assert(3 * kPerStage < 64, "vmcnt counts to 63");
  if (stages <= 0)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  else if (stages == 1)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPerStage) : "memory");
  else if (stages == 2)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kPerStage) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * kPerStage) : "memory");
}

// The task's part: its result (of one part) or its partial result. False, with
// nothing written, where something that is not finite came out
// (pf_tile_scalar then does it again).
//
// A step's softmax goes on beside the next step's scores, and that one's
// maximum beside the step's product with V: a wave has a product under way at
// nearly all times.
template <typename T, int D, int NW, int WK>
__device__ __forceinline__ bool pf_tile(const PrefillMmParams& p, const PfTask& task,
                                        const PrefillRow& r, char* lds, PfShared<NW>& sh) {
  using Shape = PfShape<T, D, NW>;
  constexpr bool F = Shape::kF32;
  constexpr int ES = Shape::kElt;
  constexpr int KTB = Shape::kStepKeys;
  constexpr int RB = Shape::kRowBytes;
  using Swz = Swizzle<RB, F>;
  constexpr int KT = KTB / WK;
  static_assert(KT % 32 == 0, "32 keys a wave at least");
  constexpr int NB = KT / 32;             // key blocks of a wave's step
  constexpr int KS = F ? D / 8 : D / 16;  // 16-byte operands over the dims of a score
  constexpr int DB = (D + 31) / 32;       // blocks of output dims
  constexpr int CPR = RB / 16;            // 16-byte chunks of a row
  constexpr int LOADS = KTB * CPR / kWave;   // per step, of K and of V
  constexpr int NJ = (LOADS + NW - 1) / NW;  // per wave
  constexpr int kScores = KS * NB;                            // products of a step with K
  constexpr int kValues = F ? DB * 4 * NB : DB * 2 * NB;      // and with V
  constexpr int AHEAD = std::min(kReadAhead, std::min(kScores, kValues));
  constexpr float kShift = std::is_same<T, F16>::value ? 7.f : 0.f;
  const PrefillArgs& a = p.a;

  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = uniform(tid / kWave);
  const int wq = wave / WK, wk = wave % WK;
  const int col = lane & 31, half = lane >> 5;
  const int rows = r.nq * p.G;
  const int wrow = task.row0 + 32 * wq;  // the wave's first query row
  const bool works = wrow < rows;
  const int rho = min(wrow + col, rows - 1);  // this lane's
  const int tok = rho / p.G;
  const int head = task.kvh * p.G + (rho - tok * p.G);
  const int vis = last_key(a, r, tok);
  const int vis_lo = uniform(vis);
  const int vis_hi = uniform(last_key(a, r, min(wrow + 31, rows - 1) / p.G));
  const int s_from = uniform(min(task.steps, task.part * task.per));
  const int s_to = uniform(min(task.steps, s_from + task.per));
  // the steps of which this wave's rows see a key: [s_from, w_to)
  const int w_to = uniform(works && vis_hi >= wk * KT ? min(s_to, (vis_hi - wk * KT) / KTB + 1) : 0);

  // Q: the row's chunks 2 ks + half of 16 bytes
  u32x4 q[KS];
  {
    const char* qp = static_cast<const char*>(a.q) +
                     ((int64_t)(r.q0 + tok) * a.q_st + (int64_t)head * a.q_sh) * ES + 16 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
  }

  // Where the part's keys lie: a table in LDS of the byte offset of every
  // 2^shift keys (a run inside a block and a step) from the first's, K's and,
  // where its strides are others, V's.
  const uint32_t lds0 = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
  const int stages = p.stages;
  int64_t* table = reinterpret_cast<int64_t*>(lds + stages * Shape::kStageBytes + Shape::kPad);
  const int end_key = uniform(min(s_to * KTB, r.nk) - 1);  // the part's last key
  const int shift = p.run_shift;
  const int run0 = uniform((s_from * KTB) >> shift);
  const int v_table = a.k_sb == a.v_sb && a.k_st == a.v_st ? 0 : p.table_room;
  bool bad = false;
  // the row's blocks that these tokens do not see: a bad id there makes the
  // row NaN too, in the first part's name
  if (a.bt != nullptr && task.part == 0)
    for (int64_t b = task.seen / a.BS + tid; b * a.BS < r.nk; b += Shape::kThreads)
      bad |= (uint32_t)a.bt[(int64_t)task.i * a.bt_stride + b] >= (uint64_t)a.num_blocks;
  if (s_from < s_to) {
    const int count = (end_key >> shift) - run0 + 1;
    for (int x = tid; x < count; x += Shape::kThreads) {
      const int key = (run0 + x) << shift;
      int64_t id = r.k0 + key, in = 0;
      if (a.bt != nullptr) {
        id = a.bt[(int64_t)task.i * a.bt_stride + key / a.BS];
        in = key % a.BS;
        const bool ok = (uint32_t)id < (uint64_t)a.num_blocks;
        bad |= !ok;
        id = ok ? id : 0;
      }
      table[x] = (id * a.k_sb + in * a.k_st) * ES;
      if (v_table != 0) table[x + v_table] = (id * a.v_sb + in * a.v_st) * ES;
    }
    __syncthreads();
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] ^= p.q_flip;
  // Loads of a stage, a step's V and the next one's K, 16 bytes a lane. What
  // lies inside the runs is the same in every step and, where the rows of two
  // loads of a lane lie whole runs apart, in every load: the loads take their
  // runs' offsets, looked up a step ahead. Not so the part's last step, whose
  // keys past the end are its last key: it looks all up at once.
  constexpr int NP = NW * kWave % (CPR * kMostRun) == 0 ? 1 : NJ;
  const char *kptr[NP], *vptr[NP];
  const int in_run = (1 << shift) - 1;
  auto row_at = [&](int j, int ln) { return ((j * NW + wave) * kWave + ln) / CPR % KTB; };
  auto chunk_at = [&](int j, int ln) { return ((j * NW + wave) * kWave + ln) % CPR; };
  auto row_of = [&](int j) { return row_at(j, lane); };
  auto chunk_of = [&](int j) { return chunk_at(j, lane); };
  auto place = [&](const void* base, int64_t sh_, int64_t st_, int key, int chunk) {
    return static_cast<const char*>(base) +
           ((int64_t)task.kvh * sh_ + (int64_t)(key & in_run) * st_) * ES + 16 * chunk;
  };
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    kptr[j] = place(a.k, a.k_sh, a.k_st, row_of(j), chunk_of(j) ^ Swz::k(row_of(j)));
    vptr[j] = place(a.v, a.v_sh, a.v_st, row_of(j), chunk_of(j) ^ Swz::v(row_of(j)));
  }
  auto lds_of = [&](int stage, int y) {
    return uniform(lds0 + stage * Shape::kStageBytes + (y / 2 * NW + wave) * (kWave * 16) +
                   (y % 2 == 0 ? 0 : KTB * RB));
  };
  auto has_load = [&](int j) { return LOADS % NW == 0 || j * NW + wave < LOADS; };
  int64_t krun[NJ], vrun[NJ];
  // looks the runs of stage `step` up
  auto locate = [&](int step) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      krun[j] = table[(((step + 1) * KTB + row_of(j)) >> shift) - run0];
      vrun[j] = table[((step * KTB + row_of(j)) >> shift) - run0 + v_table];
    }
  };
  // load y (of K and of V in turn) of the stage that was looked up
  auto load = [&](int stage, int y) {
    const int j = y / 2;
    if (!has_load(j)) return;
    load_lds16(y % 2 == 0 ? kptr[j % NP] + krun[j] : vptr[j % NP] + vrun[j], lds_of(stage, y));
  };
  auto load_last = [&](int stage, int step, int kinds) {
    int ln = lane;
    stay(ln);  // (nothing of this is to be kept in registers over the loop)
#pragma unroll
    for (int y = 0; y < 2 * NJ; y += kinds) {
      const int j = y / 2;
      if (!has_load(j)) continue;
      const bool is_k = y % 2 == 0;
      const int row = row_at(j, ln), c = chunk_at(j, ln);
      const int key = min((is_k ? step + 1 : step) * KTB + row, end_key);
      const int64_t run = table[(key >> shift) - run0 + (is_k ? 0 : v_table)];
      const char* from = is_k ? place(a.k, a.k_sh, a.k_st, key, c ^ Swz::k(row))
                              : place(a.v, a.v_sh, a.v_st, key, c ^ Swz::v(row));
      load_lds16(from + run, lds_of(stage, y));
    }
  };
  // whether stage `step` holds whole steps
  auto whole = [&](int step) { return (step + 2) * KTB - 1 <= end_key; };

  // addresses inside a stage: K row col of the wave's block 0; V: this lane's
  // part of the transposing read (row 4 half + (lane % 16) / 4 of 16 keys,
  // dims 16 ((lane / 16) % 2) + 4 (lane % 4))
  const int krow = wk * KT + col;
  const int vrow = wk * KT + 4 * half + ((lane & 15) >> 2);
  const int vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  f32x16 acc[DB];
  float m = neg_inf(), l = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;

  f32x16 s[NB];   // the step's weights' exponents, then (fp32) its weights
  f32x16 sn[NB];  // the next step's scores
  f32x16 sw[NB];  // the next step's exponents, on their way to s
  // scores of the K in `ks_lds`, with `beside` going on
  u32x4 buf[AHEAD];
  auto scores = [&](const char* ks_lds, auto&& beside, auto&& next) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) sn[nb][e] = 0.f;
    products<kScores, AHEAD, 0>(
        buf, false,
        [&](int x) {
          const int row = krow + 32 * (x % NB), c = 2 * (x / NB) + half;
          return *reinterpret_cast<const u32x4*>(ks_lds + row * RB + 16 * (c ^ Swz::k(row)));
        },
        [&](int x, const u32x4& kf) {
          if constexpr (F) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              sn[x % NB] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                  __uint_as_float(kf[e]), __uint_as_float(q[x / NB][e]), sn[x % NB], 0, 0, 0);
          } else {
            sn[x % NB] = mfma32<T>(kf, q[x / NB], sn[x % NB]);
          }
        },
        beside, next);
  };
  // operand x of the product with the V in `vs_lds`: 16 keys' (fp32: keys
  // 8 g + 4 half .. + 3, one dim a lane)
  auto value = [&](const char* vs_lds, int x) {
    u32x4 v;
    if constexpr (F) {
      const char* pv = vs_lds + (wk * KT + 8 * (x / DB) + 4 * half) * RB + (32 * (x % DB) + col) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const uint32_t*>(pv + e * RB);
    } else {
      const int r0 = vrow + 16 * (x / DB);  // and 8 rows on
      const int d = 32 * (x % DB) + vdim;
      const char* p0 = vs_lds + r0 * RB + (((d >> 3) ^ Swz::v(r0)) << 4) + (d & 7) * 2;
      const char* p1 = vs_lds + (r0 + 8) * RB + (((d >> 3) ^ Swz::v(r0 + 8)) << 4) + (d & 7) * 2;
      const uint2 v0 =
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0));
      const uint2 v1 =
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p1));
      v = u32x4{v0.x, v0.y, v1.x, v1.y};
    }
    return v;
  };
  auto mask = [&](int step) {
    const int key0 = step * KTB + wk * KT;
    if (key0 + KT - 1 <= vis_lo) return;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = key0 + 32 * nb + 8 * (e / 4) + 4 * half + e % 4;
        sn[nb][e] = key <= vis ? sn[nb][e] : neg_inf();
      }
  };
  float ms = -kShift;  // what the exponents are relative to: the running maximum, less the shift
  float top = 0.f;
  // part x of n of the next step's exponents, by the maximum so far, and their
  // own maximum
  auto take = [&](int x, int n) {
#pragma unroll
    for (int e = 16 * NB * x / n; e < 16 * NB * (x + 1) / n; ++e) {
      float y = fmaf(sn[e / 16][e % 16], p.scale_log2, -ms);
      stay(y);
      top = e == 0 ? y : fmaxf(top, y);
      sw[e / 16][e % 16] = y;
    }
    stay(top);
  };
  // the running maximum, raised where they pass it by too much (seldom: only
  // then are the exponents moved, and what is summed rescaled)
  auto raise_max = [&]() {
    top = xor_max<32>(top);
    // (the first keys raise it whatever they score; -inf is none)
    const bool raise = top > (m == neg_inf() ? neg_inf() : kLazyRescale + kShift);
    if (__ballot(raise) != 0) {
      const float mn = raise ? top + ms : m;
      const float alpha = raise ? fast_exp2(m - mn) : 1.f;
      const float by = raise ? (mn - kShift) - ms : 0.f;  // the exponents' move
      m = mn;
      ms = raise ? mn - kShift : ms;
      l *= alpha;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) sw[nb][e] -= by;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[db][e] *= alpha;
    }
  };
  u32x4 pf[F ? 1 : 2 * NB];
  float sum[2];
  // pair x of the step's weights
  auto weights = [&](int x) {
    const int nb = x / 8, e = x % 8 * 2;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float y = s[nb][e + k];
      stay(y);
      y = fast_exp2(y);
      sum[k] += y;
      if constexpr (F) stay(y);
      s[nb][e + k] = y;
    }
    if constexpr (!F) {
      uint32_t w = pack2<T>(s[nb][e], s[nb][e + 1]);
      stay(w);
      pf[2 * nb + e / 8][e % 8 / 2] = w;
    }
    stay(sum[0]);
    stay(sum[1]);
  };
  constexpr int kPairs = 8 * NB;

  constexpr int kPerStage = 2 * (LOADS / NW);
  int rd = 0, wr = stages - 1;  // the step's stage, and the one to load
  if (s_from < s_to) {
    // the first step's K, in the place of the stage that is loaded last
    load_last(wr, s_from - 1, 2);
    const int ahead = min(stages - 1, s_to - s_from);
    for (int x = 0; x < ahead; ++x) load_last(x, s_from + x, 1);
    if (whole(s_from + stages - 1)) locate(s_from + stages - 1);
    wait_loads<kPerStage>(ahead);
    __syncthreads();
    if (s_from < w_to) {
      scores(lds + wr * Shape::kStageBytes, [](int) {}, [&](int) { return u32x4{0, 0, 0, 0}; });
      mask(s_from);
      take(0, 1);
      raise_max();
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = sw[nb];
    }
  }
  for (int step = s_from; step < s_to; ++step) {
    wait_loads<kPerStage>(min(stages - 2, s_to - 1 - step));
    __syncthreads();
    const char* kn_lds = lds + rd * Shape::kStageBytes;
    const char* vs_lds = kn_lds + KTB * RB;
    const bool more = step + 1 < w_to;
    const bool beside = more && whole(step + stages - 1);
    if (!beside && step + stages - 1 < s_to) load_last(wr, step + stages - 1, 1);
    if (step < w_to) {
      sum[0] = sum[1] = 0.f;
      auto next_value = [&](int y) { return value(vs_lds, y); };
      auto some_weights = [&](int x) {
#pragma unroll
        for (int y = kPairs * x / kScores; y < kPairs * (x + 1) / kScores; ++y) weights(y);
      };
      if (beside) {
        scores(
            kn_lds,
            [&](int x) {
#pragma unroll
              for (int y = 2 * NJ * x / kScores; y < 2 * NJ * (x + 1) / kScores; ++y) load(wr, y);
              some_weights(x);
            },
            next_value);
        mask(step + 1);
      } else if (more) {
        scores(kn_lds, some_weights, next_value);
        mask(step + 1);
      } else {
#pragma unroll
        for (int y = 0; y < kPairs; ++y) weights(y);
#pragma unroll
        for (int y = 0; y < AHEAD; ++y) buf[(kScores + y) % AHEAD] = next_value(y);
      }
      l += sum[0] + sum[1];
      if (whole(step + stages)) locate(step + stages);
      // (scores that are not there are taken over to no use)
      products<kValues, AHEAD, kScores % AHEAD>(
          buf, true, next_value,
          [&](int x, const u32x4& vf) {
            if constexpr (F) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[x % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                    __uint_as_float(vf[e]), s[x / DB / 4][4 * (x / DB % 4) + e], acc[x % DB], 0, 0, 0);
            } else {
              acc[x % DB] = mfma32<T>(vf, pf[x / DB], acc[x % DB]);
            }
          },
          [&](int x) { take(x, kValues); }, [&](int) { return u32x4{0, 0, 0, 0}; });
      if (more) raise_max();
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = sw[nb];
    } else if (whole(step + stages)) {
      locate(step + stages);
    }
    rd = rd + 1 == stages ? 0 : rd + 1;
    wr = wr + 1 == stages ? 0 : wr + 1;
  }
  // anything that is not finite came from the inputs, or from values that a
  // row must not see
  bool odd = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (32 * db + 8 * (e / 4) < D) odd |= !(fabsf(acc[db][e]) < __builtin_huge_valf());
  odd = odd && works;
  if (__syncthreads_or(odd || bad) != 0) {
    if (__syncthreads_or(odd) != 0) return false;
    bad = __syncthreads_or(bad) != 0;  // a block outside the cache
  }

  l = xor_sum<32>(l);
  // ---- merge of the key waves
  if constexpr (WK > 1) {
    static_assert(WK == 2, "two key waves");
    static_assert(Shape::kMergeBytes <= 2 * Shape::kStageBytes, "the merge fits the stages");
    constexpr int kAcc = DB * 16 * kWave;  // floats of a wave
    float* buf = reinterpret_cast<float*>(lds) + wq * kAcc;
    if (half == 0) {
      sh.ml[wave][0][col] = m;
      sh.ml[wave][1][col] = l;
    }
    __syncthreads();
    const float m2 = sh.ml[wave ^ 1][0][col], l2 = sh.ml[wave ^ 1][1][col];
    const float mn = fmaxf(m, m2);
    const float base = mn == neg_inf() ? 0.f : mn;
    const float f = fast_exp2(m - base), f2 = fast_exp2(m2 - base);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] *= f;
    l = l * f + l2 * f2;
    m = mn;
    if (wk == 1 && works) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) buf[(db * 16 + e) * kWave + lane] = acc[db][e];
    }
    __syncthreads();
    if (wk == 1) return true;
    if (works) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[db][e] += buf[(db * 16 + e) * kWave + lane];
    }
  }

  if (!works || wrow + col >= rows) return true;
  const float mref = m - kShift;  // (the sums' reference)
  if (task.parts > 1) {
    const PfPartial part(p, task, r, task.part);
    const int x = 32 * wq + col;
    if (half == 0) part.store_ml(x, bad ? qnan() : l == 0.f ? neg_inf() : mref, bad ? qnan() : l);
    if (l == 0.f && !bad) return true;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (32 * db + 8 * g >= D) continue;
        const float y[4] = {acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
        part.store4(part.at(D, x, 8 * db + 2 * g + half), y);
      }
    return true;
  }
  const int t = r.q0 + tok;
  const float inv = bad ? qnan() : l == 0.f ? 0.f : 1.f / l;
  if (half == 0)
    a.lse[(int64_t)head * a.lse_sh + t] =
        bad ? qnan() : l == 0.f ? neg_inf() : (mref + fast_log2(l)) * kLn2;
  const int64_t ob = (int64_t)t * a.out_st + (int64_t)head * a.out_sh + 4 * half;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (32 * db + 8 * g >= D) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = acc[db][4 * g + e] * inv;
      pf_store4<T>(a, ob + 32 * db + 8 * g, y);
    }
  return true;
}

// The task of pf_tile on the vector ALUs, key by key: a row takes in what it
// sees and nothing else. KTB: keys of a step.
template <int D, int KTB, int NW>
__device__ __forceinline__ void pf_tile_scalar(const PrefillMmParams& p, const PfTask& task,
                                               const PrefillRow& r) {
  const PrefillArgs& a = p.a;
  constexpr int kPerLane = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave;
  const int end = min(task.row0 + task.count, r.nq * p.G);
  const int from = min(task.steps, task.part * task.per) * KTB;
  const int to = min(min(task.steps, task.part * task.per + task.per) * KTB, r.nk);
  // (the tile's own attempt may have met a bad block id: it is looked up again)
  bool bad = false;
  if (a.bt != nullptr)
    for (int64_t b = from / a.BS + lane; b * a.BS < (task.part == 0 ? r.nk : to); b += kWave)
      bad |= (uint32_t)a.bt[(int64_t)task.i * a.bt_stride + b] >= (uint64_t)a.num_blocks;
  bad = __ballot(bad) != 0;
  const PfPartial part(p, task, r, task.part);
  for (int rho = task.row0 + (int)threadIdx.x / kWave; rho < end; rho += NW) {
    const int tok = rho / p.G, head = task.kvh * p.G + rho % p.G, t = r.q0 + tok;
    float m = neg_inf(), l = 0.f, acc[kPerLane];
    scalar_attention(a, task.i, r, t, head, from, bad ? from : min(to, last_key(a, r, tok) + 1), m,
                     l, acc);
    if (bad) {
      m = l = qnan();
#pragma unroll
      for (int x = 0; x < kPerLane; ++x) acc[x] = qnan();
    }
    if (task.parts > 1) {
      const int x = rho - task.row0;
      if (lane == 0) part.store_ml(x, m * kLog2e, l);
#pragma unroll
      for (int y = 0; y < kPerLane; ++y) {
        const int d = lane + y * kWave;
        if (d < D) part.store1(part.at(D, x, d / 4) + d % 4 * 4, acc[y]);
      }
    } else {
      scalar_store(a, t, head, m, l, acc);
    }
  }
}

// Joins the parts of the task's rows, in order whichever came last: a wave
// takes 32 rows and 32 dims at a time, kInFlight parts' read together (each
// round is a trip past the L2).
template <typename T, int D, int NW, int kInFlight>
__device__ __forceinline__ void pf_merge(const PrefillMmParams& p, const PfTask& task,
                                         const PrefillRow& r) {
  constexpr int DB = (D + 31) / 32;
  const PrefillArgs& a = p.a;
  const int lane = threadIdx.x % kWave, col = lane & 31, half = lane >> 5;
  const int n = min(task.count, r.nq * p.G - task.row0);
  const int pieces = (n + 31) / 32 * DB;
  for (int piece = uniform((int)threadIdx.x / kWave); piece < pieces; piece += NW) {
    const int x = piece / DB * 32 + col, db = piece % DB;
    if (x >= n) continue;
    float m = neg_inf(), l = 0.f, acc[4][4] = {};
    for (int k0 = 0; k0 < task.parts; k0 += kInFlight) {
      uint2_v ml[kInFlight];
      u32x4 o[kInFlight][4];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        // a part past the last reads the last one again, to no effect
        const PfPartial part(p, task, r, min(k0 + u, task.parts - 1));
        ml[u] = __builtin_amdgcn_raw_buffer_load_b64(part.ml, x * 8, 0, kAgentScope);
#pragma unroll
        for (int g = 0; g < 4; ++g)  // (dims past D read 0, or another row's)
          o[u][g] = __builtin_amdgcn_raw_buffer_load_b128(
              part.o, part.at(D, x, 8 * db + 2 * g + half), 0, kAgentScope);
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const float mp = __uint_as_float(ml[u][0]), lp = __uint_as_float(ml[u][1]);
        // (a part without keys has no sums; what lies there is not read as one)
        if (k0 + u >= task.parts || lp == 0.f) continue;
        const float mn = fmaxf(m, mp);
        const float base = mn == neg_inf() ? 0.f : mn;
        const float f = fast_exp2(m - base), w = fast_exp2(mp - base);
        m = mn;
        l = l * f + lp * w;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[g][e] = acc[g][e] * f + __uint_as_float(o[u][g][e]) * w;
      }
    }
    const int rho = task.row0 + x, tok = rho / p.G;
    const int head = task.kvh * p.G + (rho - tok * p.G);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t t = r.q0 + tok;
    if (db == 0 && half == 0)
      a.lse[(int64_t)head * a.lse_sh + t] = l == 0.f ? neg_inf() : (m + fast_log2(l)) * kLn2;
    const int64_t ob = t * a.out_st + (int64_t)head * a.out_sh + 32 * db + 4 * half;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (D % 32 != 0 && 32 * db + 8 * g >= D) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[g][e] *= inv;
      pf_store4<T>(a, ob + 8 * g, acc[g]);
    }
  }
}

// NaN (a range error) for `count` rows from row0 on of row r and this kv head.
template <int NW>
__device__ __forceinline__ void pf_fill_nan(const PrefillMmParams& p, const PrefillRow& r, int row0,
                                            int64_t count, int kvh) {
  const PrefillArgs& a = p.a;
  const int64_t end = min(row0 + count, (int64_t)r.nq * p.G);
  for (int64_t rho = row0 + (int)threadIdx.x / kWave; rho < end; rho += NW) {
    const int head = kvh * p.G + (int)(rho % p.G), lane = threadIdx.x % kWave;
    const int64_t t = r.q0 + rho / p.G;
    for (int d = lane; d < a.D; d += kWave)
      store_elem(a.out, t * a.out_st + (int64_t)head * a.out_sh + d, a.out_dt, qnan());
    if (lane == 0) a.lse[(int64_t)head * a.lse_sh + t] = qnan();
  }
}

// A workgroup's task by its index: A tasks first (their tiles from the last to
// the first: under a causal mask a row's last tiles have the most keys), kv
// heads fastest, so that an XCD keeps to few of them and a kv head's keys stay
// in its L2. A tile's keys are cut into parts of a fixed number of steps; the
// grid holds as many parts as the longest row may have, and those that a tile
// does not have end at once.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * kWave, (PfShape<T, D, NW>::kWavesPerSimd)) void
prefill_mm_kernel(PrefillMmParams p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ PfShared<NW> sh;
  using Shape = PfShape<T, D, NW>;
  constexpr int KTB = Shape::kStepKeys;
  const PrefillArgs& a = p.a;
  PfTask task{};
  int b = blockIdx.x;
  task.kvh = b % a.KVH;
  b /= a.KVH;
  const int tasks_a = p.plan.tiles_a * p.plan.parts_a;
  const bool is_a = b < tasks_a;
  int tile = 0, slot = 0;
  PrefillRow r;
  if (is_a) {
    task.part = b / p.plan.tiles_a;
    task.per = p.plan.per_a;
    slot = b % p.plan.tiles_a;
    tile = p.plan.tiles_a - 1 - slot;
    if (a.n > 1) {
      // the row that holds A tile `tile`: tiles of the rows ahead, 64 rows a round
      const int lane = threadIdx.x % kWave;
      bool found = false;
      for (int c = 0; c < a.n && !found; c += kWave) {
        int tiles = 0;
        PrefillRow x{};
        if (c + lane < a.n) {
          x = prefill_row(a, c + lane);
          const int64_t rows = (int64_t)x.nq * p.G;
          if (p.plan.rows_b == 0 || rows > kRowsB)
            tiles = (int)((rows + Shape::kRowsA - 1) / Shape::kRowsA);
        }
        int upto = tiles;
        for (int d = 1; d < kWave; d <<= 1) {
          const int o = __shfl_up(upto, d, kWave);
          if (lane >= d) upto += o;
        }
        const int total = __shfl(upto, kWave - 1, kWave);
        if (tile < total) {
          const uint64_t past = __ballot(upto > tile);
          const int w = __builtin_ctzll(past);
          task.i = c + w;
          tile -= __shfl(upto, w, kWave) - __shfl(tiles, w, kWave);
          r = PrefillRow{__shfl(x.q0, w, kWave), __shfl(x.nq, w, kWave), __shfl(x.k0, w, kWave),
                         __shfl(x.nk, w, kWave), __shfl((int)x.bad, w, kWave) != 0};
          found = true;
        } else {
          tile -= total;
        }
      }
      if (!found) return;
    } else {
      r = prefill_row(a, 0);
    }
    task.count = Shape::kRowsA;
  } else {
    b -= tasks_a;
    task.part = b / p.plan.rows_b;
    task.per = p.plan.per_b;
    task.i = b % p.plan.rows_b;
    slot = p.plan.tiles_a + task.i;
    task.count = kRowsB;
    r = prefill_row(a, task.i);
  }
  task.i = uniform(task.i);
  task.row0 = uniform(tile) * task.count;
  r.q0 = uniform(r.q0);
  r.nq = uniform(r.nq);
  r.k0 = uniform(r.k0);
  r.nk = uniform(r.nk);
  const int64_t rows = (int64_t)r.nq * p.G;
  if (task.row0 >= rows) return;
  if (!is_a && rows > kRowsB) {
    // an A row, or (without A tasks) more tokens than the call said: all of it
    if (p.plan.tiles_a == 0 && task.part == 0) pf_fill_nan<NW>(p, r, 0, rows, task.kvh);
    return;
  }
  if (r.bad) {
    if (task.part == 0) pf_fill_nan<NW>(p, r, task.row0, task.count, task.kvh);
    return;
  }
  task.seen = max(0, last_key(a, r, ((int)min((int64_t)task.row0 + task.count, rows) - 1) / p.G) + 1);
  task.steps = (task.seen + KTB - 1) / KTB;
  task.parts = max(1, (task.steps + task.per - 1) / task.per);
  if (task.part >= task.parts) return;
  uint64_t* counter = p.counters + ((int64_t)slot * a.KVH + task.kvh) * p.counter_stride;
  if (task.parts > 1 && threadIdx.x == 0)
    __hip_atomic_fetch_max(counter, p.launch, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  constexpr int kWk = KTB / 32;  // key waves of a B tile
  const bool done = is_a ? pf_tile<T, D, NW, 1>(p, task, r, lds, sh)
                         : pf_tile<T, D, NW, kWk>(p, task, r, lds, sh);
  if (!done) pf_tile_scalar<D, KTB, NW>(p, task, r);
  if (task.parts == 1) return;
  // The last part to be written joins them all: its stores done, each part
  // counts itself (a count starts anew with every launch: the launch's number
  // stands above it, as in the decode kernels).
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  __syncthreads();
  if (threadIdx.x == 0) {
    constexpr uint64_t kCount = (1ull << kLaunchBits) - 1;
    const uint64_t before =
        __hip_atomic_fetch_add(counter, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = (int)(before & kCount) == task.parts - 1;
    if (last)
      __hip_atomic_store(counter, before & ~kCount, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sh.last = last ? 1 : 0;
  }
  __syncthreads();
  const bool last = uniform(sh.last) != 0;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");  // no part is read before
  if (last && task.parts <= 2) {
    pf_merge<T, D, NW, 2>(p, task, r);
  } else if (last) {
    pf_merge<T, D, NW, 8>(p, task, r);
  }
}

template <typename T, int D, int NW>
hipError_t launch_d(PrefillMmParams p, hipStream_t s) {
  using Shape = PfShape<T, D, NW>;
  const auto kernel = prefill_mm_kernel<T, D, NW>;
  constexpr int kStatic = 4096;  // PfShared, and what the compiler adds
  constexpr int kMost = 160 * 1024 - kStatic;
  static const hipError_t set = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (set != hipSuccess) return set;
  // two workgroups of four waves share a CU where two stages of both fit (and
  // the registers of both)
  const int tail = Shape::kPad + 8 * p.table_room * (p.a.k_sb == p.a.v_sb && p.a.k_st == p.a.v_st ? 1 : 2);
  const int half = (80 * 1024 - kStatic - tail) / Shape::kStageBytes;
  const bool two = NW == 4 && Shape::kWavesPerSimd == 2 && half >= 2 && !p.alone;
  const int per = std::max(p.plan.tiles_a > 0 ? p.plan.per_a : 0, p.plan.rows_b > 0 ? p.plan.per_b : 0);
  p.stages = std::min(std::min(4, std::max(2, per + 1)), two ? half : (kMost - tail) / Shape::kStageBytes);
  if (p.stages < 2) return hipErrorInvalidValue;  // (table_room in prefill.hip leaves room for two)
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.grid), dim3(Shape::kThreads),
                     p.stages * Shape::kStageBytes + tail, s, p);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_q(const PrefillMmParams& p, hipStream_t s) {
  if constexpr (D <= 128)
    if (p.plan.waves == 8) return launch_d<T, D, 8>(p, s);
  return launch_d<T, D, 4>(p, s);
}

template <typename T>
int launch_prefill_mm(const PrefillMmParams& p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  switch (p.a.D) {
    case 32: e = launch_q<T, 32>(p, s); break;
    case 48: e = launch_q<T, 48>(p, s); break;
    case 64: e = launch_q<T, 64>(p, s); break;
    case 80: e = launch_q<T, 80>(p, s); break;
    case 96: e = launch_q<T, 96>(p, s); break;
    case 112: e = launch_q<T, 112>(p, s); break;
    case 128: e = launch_q<T, 128>(p, s); break;
    case 256: e = launch_q<T, 256>(p, s); break;
  }
  return e == hipSuccess ? FD_OK : hip_error(e, "prefill_mm_kernel launch");
}

}  // namespace

}  // namespace fd
