// Attention of packed query tokens with both products on the matrix cores,
// instantiated per type by prefill_mm_f16.hip, prefill_mm_bf16.hip and
// prefill_mm_f32.hip.
//
// A workgroup of four waves takes a tile of query rows of one kv head and
// walks the tile's keys. Query rows are (token, head of the kv head's group)
// pairs, so grouped-query heads share every K and V read and a few tokens of
// many heads fill a tile as well as many tokens of one. Waves stand WQ x WK:
// WQ times 32 rows, WK parts of each step's keys (A: 4 x 1 on 64 keys a step;
// B: 2 x 2 on 32 each, for rows that bring few tokens and are bound by the
// read of K and V).
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
// K and V go to LDS by global_load_lds (16 bytes a lane, no registers), two
// stages: step t + 1 is under way while t is computed, one barrier a step. The
// loads land in order of lanes, so the bank swizzle is in the address that a
// lane reads: LDS slot c of a K row holds chunk c ^ swizzle_k(row), of a V row
// chunk c ^ swizzle_v(row); K is read 16 rows x 16 bytes at a time, V 4 rows x
// 64 bytes.
//
// Keys that no row of a wave sees are skipped, steps that some row sees in
// part are masked (a key against the row's last). What the masked V rows hold
// does not matter as long as it is finite (weight 0); where a result is not
// finite, the workgroup does its tile again with every masked step's
// infinities and NaNs taken out of V and put back only into rows that give
// them weight.
#pragma once

#include <type_traits>

#include "prefill_mm.h"

namespace fd {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_ptr;

constexpr int kPfWaves = 4;
constexpr int kPfThreads = kPfWaves * kWave;
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

template <typename T, int D>
struct PfShape {
  static constexpr bool kF32 = std::is_same<T, F32>::value;
  static constexpr int kElt = kF32 ? 4 : 2;
  static constexpr int kStepKeys = kElt * D <= 256 ? 64 : 32;  // keys of a step
  static constexpr int kRowBytes = D * kElt;
  // waves a SIMD holds by the registers that a wave needs
  static constexpr int kWavesPerSimd = kF32 && D > 128 ? 1 : 2;
  static constexpr int kStageBytes = kStepKeys * kRowBytes;  // of K, and of V
  // the merge of a B tile's two key waves: fp32 accumulators of half the waves
  static constexpr int kMergeBytes = 2 * ((D + 31) / 32 * 32) * 32 * 4;
  static constexpr int kStages = 4 * kStageBytes + 32 * kElt;  // (reads past D in the last row)
  static constexpr int kLds = kStages > kMergeBytes ? kStages : kMergeBytes;
};

// kCount products, each behind the LDS reads of the product kAhead further on:
// read(x) gives product x's operand, use(x, operand) computes it. In this
// order by force: left to itself the compiler reads each operand right ahead
// of its product, which then waits for it.
template <int kCount, int kAhead, typename R, typename U>
__device__ __forceinline__ void read_ahead(R&& read, U&& use) {
  u32x4 buf[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead && x < kCount; ++x) buf[x] = read(x);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int x = 0; x < kCount; ++x) {
    use(x, buf[x % kAhead]);
    if (x + kAhead < kCount) buf[x % kAhead] = read(x + kAhead);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The first lane's value, known to be every lane's.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

struct PfShared {
  float ml[kPfWaves][2][32];
};

// One tile: rows [row0, row0 + 32 WQ) of row r's nq * G, part `part` of its
// keys. False, with nothing written, where something that is not finite came
// out (pf_tile_scalar then does the tile again).
template <typename T, int D, int WQ, int WK>
__device__ __forceinline__ bool pf_tile(const PrefillMmParams& p, int i, const PrefillRow& r,
                                        int row0, int kvh, int part, int parts, char* lds,
                                        PfShared& sh, int tid) {
  static_assert(WQ * WK == kPfWaves, "four waves");
  constexpr bool F = PfShape<T, D>::kF32;
  constexpr int ES = PfShape<T, D>::kElt;
  constexpr int KTB = PfShape<T, D>::kStepKeys;
  using Swz = Swizzle<PfShape<T, D>::kRowBytes, F>;
  constexpr int KT = KTB / WK;
  static_assert(KT % 32 == 0, "32 keys a wave at least");
  constexpr int NB = KT / 32;         // key blocks of a wave's step
  constexpr int KS = F ? D / 8 : D / 16;  // 16-byte operands over the dims of a score
  constexpr int DB = (D + 31) / 32;   // blocks of output dims
  constexpr int CPR = D * ES / 16;    // 16-byte chunks of a row
  constexpr int LOADS = KTB * CPR / kWave;                       // per step, of K and of V
  constexpr int NJ = (LOADS + kPfWaves - 1) / kPfWaves;          // per wave
  constexpr float kShift = std::is_same<T, F16>::value ? 7.f : 0.f;
  const PrefillArgs& a = p.a;

  const int lane = tid % kWave;
  const int wave = uniform(tid / kWave);
  const int wq = wave / WK, wk = wave % WK;
  const int col = lane & 31, half = lane >> 5;
  const int rows = r.nq * p.G;
  const int wrow = row0 + 32 * wq;    // the wave's first query row
  const bool works = wrow < rows;
  const int rho = min(wrow + col, rows - 1);
  const int tok = rho / p.G;
  const int head = kvh * p.G + (rho - tok * p.G);
  const int vis = last_key(a, r, tok);
  const int vis_lo = uniform(vis);
  const int vis_hi = uniform(last_key(a, r, min(wrow + 31, rows - 1) / p.G));
  // the tile's keys and this part's share of them, in whole steps
  const int all = last_key(a, r, (min(row0 + 32 * WQ, rows) - 1) / p.G) + 1;
  const int steps = (max(all, 0) + KTB - 1) / KTB;
  const int per = (steps + parts - 1) / parts;
  const int s_from = uniform(min(steps, part * per)), s_to = uniform(min(steps, s_from + per));

  // Q: row col's chunks 2 ks + half of 16 bytes
  u32x4 q[KS];
  {
    const char* qp = static_cast<const char*>(a.q) +
                     ((int64_t)(r.q0 + tok) * a.q_st + (int64_t)head * a.q_sh) * ES + 16 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
      q[ks] ^= p.q_flip;
    }
  }

  const uint32_t lds0 = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
  const char* kbase = static_cast<const char*>(a.k) + (int64_t)kvh * a.k_sh * ES;
  const char* vbase = static_cast<const char*>(a.v) + (int64_t)kvh * a.v_sh * ES;
  const bool paged = a.bt != nullptr;
  const int32_t* bt = paged ? a.bt + (int64_t)i * a.bt_stride : nullptr;
  // Where a step's keys lie: lane k of every wave looks key k up (past the
  // row's end: its last), the block id a step ahead; the loads, 16 bytes of a
  // row a lane, take their row's offset from that lane.
  bool bad = false;
  const bool one_offset = a.k_sb == a.v_sb && a.k_st == a.v_st;
  auto key_of = [&](int step) { return min(step * KTB + lane % KTB, r.nk - 1); };
  auto block_of = [&](int key) { return (int)(((uint64_t)(uint32_t)key * p.bs_magic) >> p.bs_shift); };
  int next_id = 0;
  auto fetch_id = [&](int step) {
    const int key = key_of(step);
    next_id = paged ? bt[block_of(key)] : r.k0 + key;
  };
  auto issue = [&](int step, int stage) {
    int id = next_id, in = 0;
    if (paged) {
      const bool ok = (uint32_t)id < (uint64_t)a.num_blocks;
      bad |= !ok;
      id = ok ? id : 0;
      const int key = key_of(step);
      in = key - block_of(key) * a.BS;
    }
    const int64_t ko = ((int64_t)id * a.k_sb + (int64_t)in * a.k_st) * ES;
    const int64_t vo = one_offset ? ko : ((int64_t)id * a.v_sb + (int64_t)in * a.v_st) * ES;
    auto of_lane = [](int64_t x, int src) {
      const uint32_t lo = __builtin_amdgcn_ds_bpermute(src * 4, (int)(uint32_t)x);
      const uint32_t hi = __builtin_amdgcn_ds_bpermute(src * 4, (int)(uint32_t)((uint64_t)x >> 32));
      return (int64_t)((uint64_t)hi << 32 | lo);
    };
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (LOADS % kPfWaves != 0 && j * kPfWaves + wave >= LOADS) break;
      const int u = (j * kPfWaves + wave) * kWave + lane;
      const int row = u / CPR, c = u - row * CPR;
      const int64_t kj = of_lane(ko, row);
      const int64_t vj = one_offset ? kj : of_lane(vo, row);
      const uint32_t at = lds0 + stage * 2 * PfShape<T, D>::kStageBytes +
                          (j * kPfWaves + wave) * (kWave * 16);
      load_lds16(kbase + 16 * (c ^ Swz::k(row)) + kj, at);
      load_lds16(vbase + 16 * (c ^ Swz::v(row)) + vj, at + PfShape<T, D>::kStageBytes);
    }
  };

  // addresses inside a stage: K row col of the wave's block 0; V: this lane's
  // part of the transposing read (row 4 half + (lane % 16) / 4 of 16 keys,
  // dims 16 ((lane / 16) % 2) + 4 (lane % 4))
  const int krow = wk * KT + col;
  const int vrow = wk * KT + 4 * half + ((lane & 15) >> 2);
  const int vdim = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  f32x16 acc[DB];
  float m, l;
  {
    m = neg_inf();
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] = 0.f;

    if (s_from < s_to) {
      fetch_id(s_from);
      issue(s_from, 0);
      if (s_from + 1 < s_to) fetch_id(s_from + 1);
    }
    for (int step = s_from; step < s_to; ++step) {
      const int stage = (step - s_from) & 1;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (step + 1 < s_to) {
        issue(step + 1, stage ^ 1);
        if (step + 2 < s_to) fetch_id(step + 2);
      }
      const int key0 = step * KTB + wk * KT;
      if (!works || key0 > vis_hi) continue;
      const char* ks_lds = lds + stage * 2 * PfShape<T, D>::kStageBytes;
      const char* vs_lds = ks_lds + PfShape<T, D>::kStageBytes;

      f32x16 s[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[nb][e] = 0.f;
      read_ahead<KS * NB, kReadAhead>(
          [&](int x) {
            const int row = krow + 32 * (x % NB), c = 2 * (x / NB) + half;
            return *reinterpret_cast<const u32x4*>(ks_lds + row * PfShape<T, D>::kRowBytes +
                                                   16 * (c ^ Swz::k(row)));
          },
          [&](int x, const u32x4& kf) {
            if constexpr (F) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[x % NB] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                    __uint_as_float(kf[e]), __uint_as_float(q[x / NB][e]), s[x % NB], 0, 0, 0);
            } else {
              s[x % NB] = mfma32<T>(kf, q[x / NB], s[x % NB]);
            }
          });
      const bool masked = key0 + KT - 1 > vis_lo;
      if (masked) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = key0 + 32 * nb + 8 * (e / 4) + 4 * half + e % 4;
            s[nb][e] = key <= vis ? s[nb][e] : neg_inf();
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[nb][e]);
      top = xor_max<32>(top) * p.scale_log2;
      const bool raise = top > m + kLazyRescale;  // false while both are -inf
      if (__ballot(raise) != 0) {
        const float mn = raise ? top : m;
        const float alpha = raise ? fast_exp2(m - mn) : 1.f;
        m = mn;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[db][e] *= alpha;
      }
      const float ms = (m == neg_inf() ? 0.f : m) - kShift;
      float sum = 0.f;
      if constexpr (F) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[nb][e] = fast_exp2(fmaf(s[nb][e], p.scale_log2, -ms));
            sum += s[nb][e];
          }
        l += sum;
        // operand x: keys 8 g + 4 half .. + 3 of block nb, one dim a lane
        read_ahead<DB * 4 * NB, 2>(
            [&](int x) {
              const int db = x % DB, g = x / DB;  // (g counts over the blocks)
              const char* pv = vs_lds + (wk * KT + 8 * g + 4 * half) * PfShape<T, D>::kRowBytes +
                               (32 * db + col) * 4;
              u32x4 v;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                v[e] = *reinterpret_cast<const uint32_t*>(pv + e * PfShape<T, D>::kRowBytes);
              return v;
            },
            [&](int x, const u32x4& v) {
              const int db = x % DB, g = x / DB;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                    __uint_as_float(v[e]), s[g / 4][4 * (g % 4) + e], acc[db], 0, 0, 0);
            });
      } else {
        u32x4 pf[2 * NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float pv[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            pv[e] = fast_exp2(fmaf(s[nb][e], p.scale_log2, -ms));
            sum += pv[e];
          }
#pragma unroll
          for (int e = 0; e < 16; e += 2)
            pf[2 * nb + e / 8][(e % 8) / 2] = pack2<T>(pv[e], pv[e + 1]);
        }
        l += sum;
        read_ahead<DB * 2 * NB, kReadAhead>(
            [&](int x) {
              const int r0 = vrow + 16 * (x / DB);  // and 8 rows on
              const int d = 32 * (x % DB) + vdim;
              const char* p0 = vs_lds + r0 * PfShape<T, D>::kRowBytes +
                               (((d >> 3) ^ Swz::v(r0)) << 4) + (d & 7) * 2;
              const char* p1 = vs_lds + (r0 + 8) * PfShape<T, D>::kRowBytes +
                               (((d >> 3) ^ Swz::v(r0 + 8)) << 4) + (d & 7) * 2;
              const uint2 v0 = __builtin_bit_cast(
                  uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0));
              const uint2 v1 = __builtin_bit_cast(
                  uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p1));
              return u32x4{v0.x, v0.y, v1.x, v1.y};
            },
            [&](int x, const u32x4& vf) { acc[x % DB] = mfma32<T>(vf, pf[x / DB], acc[x % DB]); });
      }
    }

    // anything that is not finite came from the inputs, or from values that a
    // row must not see
    bool odd = false;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (32 * db + 8 * (e / 4) < D) odd |= !(fabsf(acc[db][e]) < __builtin_huge_valf());
    if (__syncthreads_or(odd && works) != 0) return false;
  }
  // a block outside the cache
  bad = __syncthreads_or(bad) != 0;

  l = xor_sum<32>(l);
  // ---- merge of the key waves
  if constexpr (WK > 1) {
    static_assert(WK == 2, "two key waves");
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
    if (wk == 1) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) buf[(db * 16 + e) * kWave + lane] = acc[db][e];
    }
    __syncthreads();
    if (wk == 1) return true;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[db][e] += buf[(db * 16 + e) * kWave + lane];
  }

  if (!works || wrow + col >= rows) return true;
  const int t = r.q0 + tok;
  const float ms = m - kShift;  // (the sums' reference)
  if (parts > 1) {
    const int64_t at = (int64_t)part * a.T * a.H + (int64_t)t * a.H + head;
    if (half == 0) p.part_ml[at] = bad ? make_float2(qnan(), qnan()) : make_float2(l == 0.f ? neg_inf() : ms, l);
    if (l == 0.f && !bad) return true;
    float* po = p.part_o + at * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (32 * db + 8 * g >= D) continue;
        *reinterpret_cast<float4*>(po + 32 * db + 8 * g + 4 * half) =
            make_float4(acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]);
      }
    return true;
  }
  const float inv = bad ? qnan() : l == 0.f ? 0.f : 1.f / l;
  if (half == 0)
    a.lse[(int64_t)head * a.lse_sh + t] =
        bad ? qnan() : l == 0.f ? neg_inf() : (ms + fast_log2(l)) * kLn2;
  const int64_t ob = (int64_t)t * a.out_st + (int64_t)head * a.out_sh + 4 * half;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (32 * db + 8 * g >= D) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = l == 0.f && !bad ? 0.f : acc[db][4 * g + e] * inv;
      const int64_t o = ob + 32 * db + 8 * g;
      if (F || a.out_dt == FD_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + o) = make_float4(y[0], y[1], y[2], y[3]);
      } else if constexpr (!F) {
        uint2 u;
        u.x = to_out(T{}, y[0]) | ((uint32_t)to_out(T{}, y[1]) << 16);
        u.y = to_out(T{}, y[2]) | ((uint32_t)to_out(T{}, y[3]) << 16);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) = u;
      }
    }
  return true;
}

// The tile of pf_tile (its step's keys: STEP) on the vector ALUs, key by key:
// a row takes in what it sees and nothing else.
template <int D, int STEP>
__device__ __forceinline__ void pf_tile_scalar(const PrefillMmParams& p, int i, const PrefillRow& r,
                                               int row0, int count, int kvh, int part, int parts) {
  const PrefillArgs& a = p.a;
  constexpr int kPerLane = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave;
  const int rows = r.nq * p.G;
  const int end = min(row0 + count, rows);
  const int steps = (max(last_key(a, r, (end - 1) / p.G) + 1, 0) + STEP - 1) / STEP;
  const int per = (steps + parts - 1) / parts;
  const int from = min(steps, part * per) * STEP, to = min(steps, (part + 1) * per) * STEP;
  // (the tile's own attempt may have met a bad block id: it is looked up again)
  bool bad = false;
  if (a.bt != nullptr)
    for (int b = from / a.BS + lane; (int64_t)b * a.BS < min(to, r.nk); b += kWave)
      bad |= (uint32_t)a.bt[(int64_t)i * a.bt_stride + b] >= (uint64_t)a.num_blocks;
  bad = __ballot(bad) != 0;
  for (int rho = row0 + (int)threadIdx.x / kWave; rho < end; rho += kPfWaves) {
    const int tok = rho / p.G, head = kvh * p.G + rho % p.G, t = r.q0 + tok;
    float m = neg_inf(), l = 0.f, acc[kPerLane];
    scalar_attention(a, i, r, t, head, from, bad ? from : min(to, last_key(a, r, tok) + 1), m, l, acc);
    if (bad) m = l = acc[0] = qnan();
    if (parts > 1) {
      const int64_t at = (int64_t)part * a.T * a.H + (int64_t)t * a.H + head;
      if (lane == 0) p.part_ml[at] = make_float2(m * kLog2e, l);
      if (l == 0.f) continue;
#pragma unroll
      for (int x = 0; x < kPerLane; ++x)
        if (lane + x * kWave < D) p.part_o[at * D + lane + x * kWave] = acc[x];
    } else {
      if (bad)
        for (int x = 1; x < kPerLane; ++x) acc[x] = qnan();
      scalar_store(a, t, head, m, l, acc);
    }
  }
}

// NaN (a range error) for rows [row0, row0 + count) of row r and this kv head.
__device__ __forceinline__ void pf_fill_nan(const PrefillMmParams& p, const PrefillRow& r, int row0,
                                            int count, int kvh, int part, int parts) {
  const PrefillArgs& a = p.a;
  const int end = (int)min((int64_t)row0 + count, (int64_t)r.nq * p.G);
  for (int rho = row0 + (int)threadIdx.x / kWave; rho < end; rho += kPfWaves) {
    const int tok = rho / p.G, head = kvh * p.G + rho % p.G, lane = threadIdx.x % kWave;
    const int64_t t = r.q0 + tok;
    if (parts > 1) {
      if (lane == 0) p.part_ml[(int64_t)part * a.T * a.H + t * a.H + head] = make_float2(qnan(), qnan());
      continue;
    }
    for (int d = lane; d < a.D; d += kWave)
      store_elem(a.out, t * a.out_st + (int64_t)head * a.out_sh + d, a.out_dt, qnan());
    if (lane == 0) a.lse[(int64_t)head * a.lse_sh + t] = qnan();
  }
}

// A workgroup's task by its index: A tasks first (their tiles from the last to
// the first: under a causal mask a row's last tiles have the most keys), kv
// heads fastest, so that an XCD keeps to few of them and a kv head's keys stay
// in its L2.
template <typename T, int D>
__global__ __launch_bounds__(kPfThreads, (PfShape<T, D>::kWavesPerSimd)) void
prefill_mm_kernel(PrefillMmParams p) {
  extern __shared__ __align__(16) char lds[];
  __shared__ PfShared sh;
  const PrefillArgs& a = p.a;
  int b = blockIdx.x;
  const int kvh = b % a.KVH;
  b /= a.KVH;
  const int tasks_a = p.plan.tiles_a * p.plan.sa;
  const bool is_a = b < tasks_a;
  int part, parts, i = 0, tile = 0;
  if (is_a) {
    part = b % p.plan.sa;
    parts = p.plan.sa;
    int slot = p.plan.tiles_a - 1 - b / p.plan.sa;
    if (a.n > 1) {
      // the row that holds A tile `slot`: tiles of the rows ahead, 64 rows a round
      const int lane = threadIdx.x % kWave;
      bool found = false;
      for (int c = 0; c < a.n && !found; c += kWave) {
        int tiles = 0;
        if (c + lane < a.n) {
          const PrefillRow x = prefill_row(a, c + lane);
          const int64_t rows = (int64_t)x.nq * p.G;
          if (p.plan.rows_b == 0 || rows > kRowsB) tiles = (int)((rows + kRowsA - 1) / kRowsA);
        }
        int upto = tiles;
        for (int d = 1; d < kWave; d <<= 1) {
          const int o = __shfl_up(upto, d, kWave);
          if (lane >= d) upto += o;
        }
        const int total = __shfl(upto, kWave - 1, kWave);
        if (slot < total) {
          const uint64_t past = __ballot(upto > slot);
          const int w = __builtin_ctzll(past);
          i = c + w;
          tile = slot - (__shfl(upto, w, kWave) - __shfl(tiles, w, kWave));
          found = true;
        } else {
          slot -= total;
        }
      }
      if (!found) return;
      i = uniform(i);
      tile = uniform(tile);
    } else {
      tile = slot;
    }
  } else {
    b -= tasks_a;
    part = b % p.plan.sb;
    parts = p.plan.sb;
    i = b / p.plan.sb;
  }
  PrefillRow r = prefill_row(a, i);
  r.q0 = uniform(r.q0);
  r.nq = uniform(r.nq);
  r.k0 = uniform(r.k0);
  r.nk = uniform(r.nk);
  const int64_t rows = (int64_t)r.nq * p.G;
  const int row0 = is_a ? tile * kRowsA : 0;
  if (row0 >= rows) return;
  if (!is_a && rows > kRowsB) {
    // an A row, or (without A tasks) more tokens than the call said: all of it
    if (p.plan.tiles_a == 0) pf_fill_nan(p, r, 0, (int)rows, kvh, part, parts);
    return;
  }
  // every block of the row, whether these tokens see it or not
  bool bad = r.bad;
  if (a.bt != nullptr && part == 0 && !bad) {
    const int nb = (int)(((int64_t)r.nk + a.BS - 1) / a.BS);
    const int32_t* bt = a.bt + (int64_t)i * a.bt_stride;
    for (int x = threadIdx.x; x < nb; x += kPfThreads) bad |= (uint32_t)bt[x] >= (uint64_t)a.num_blocks;
  }
  if (__syncthreads_or(bad) != 0) {
    pf_fill_nan(p, r, row0, is_a ? kRowsA : kRowsB, kvh, part, parts);
    return;
  }
  constexpr int kWk = PfShape<T, D>::kStepKeys / 32;  // key waves of a B tile
  const int tid = threadIdx.x;
  const bool done = is_a
                        ? pf_tile<T, D, 4, 1>(p, i, r, row0, kvh, part, parts, lds, sh, tid)
                        : pf_tile<T, D, 4 / kWk, kWk>(p, i, r, row0, kvh, part, parts, lds, sh, tid);
  if (!done)
    pf_tile_scalar<D, PfShape<T, D>::kStepKeys>(p, i, r, row0, is_a ? kRowsA : kRowsB, kvh, part, parts);
}

template <typename T, int D>
hipError_t launch_d(const PrefillMmParams& p, hipStream_t s) {
  const int64_t tasks = ((int64_t)p.plan.tiles_a * p.plan.sa + (int64_t)p.plan.rows_b * p.plan.sb) * p.a.KVH;
  const auto kernel = prefill_mm_kernel<T, D>;
  constexpr int kLds = PfShape<T, D>::kLds;
  static const hipError_t set = hipFuncSetAttribute(
      reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  if (set != hipSuccess) return set;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tasks), dim3(kPfThreads), kLds, s, p);
  return hipGetLastError();
}

template <typename T>
int launch_prefill_mm(const PrefillMmParams& p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  switch (p.a.D) {
    case 32: e = launch_d<T, 32>(p, s); break;
    case 48: e = launch_d<T, 48>(p, s); break;
    case 64: e = launch_d<T, 64>(p, s); break;
    case 80: e = launch_d<T, 80>(p, s); break;
    case 96: e = launch_d<T, 96>(p, s); break;
    case 112: e = launch_d<T, 112>(p, s); break;
    case 128: e = launch_d<T, 128>(p, s); break;
    case 256: e = launch_d<T, 256>(p, s); break;
  }
  return e == hipSuccess ? FD_OK : hip_error(e, "prefill_mm_kernel launch");
}

}  // namespace

}  // namespace fd
