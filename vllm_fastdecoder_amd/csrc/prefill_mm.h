// Attention of packed query tokens on the matrix cores: the
// kernel's plan and launcher, shared by prefill.hip (planning) and the
// translation units that instantiate it per type.
#pragma once

#include "prefill.h"

namespace fd {

// How a call is cut: A tasks take kRowsA query rows of one row and kv head
// (row = token * group + head in the group), B tasks all of a row of at most
// kRowsB; each over one of sa / sb parts of the keys.
struct PrefillPlan {
  int32_t tiles_a;  // A tiles at most, over all rows (0: no A tasks)
  int32_t rows_b;   // B tasks per kv head (n, or 0: none)
  int32_t sa, sb;   // parts of the keys
  size_t workspace;
};

constexpr int kRowsA = 128;
constexpr int kRowsB = 64;

struct PrefillMmParams {
  PrefillArgs a;
  PrefillPlan plan;
  int32_t G;
  float scale_log2;      // > 0
  uint32_t q_flip;       // sign bits to flip in a word of q (a negative scale)
  uint32_t bs_magic;     // key / BS = key * bs_magic >> bs_shift, key < 2^31
  int32_t bs_shift;
  float* part_o;   // [parts][T * H][D]
  float2* part_ml; // [parts][T * H]: running maximum (log2 domain) and sum
};

PrefillPlan plan_prefill_mm(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D, int32_t max_q,
                            int64_t max_k);
int launch_prefill_mm_f16(const PrefillMmParams& p, hipStream_t s);
int launch_prefill_mm_bf16(const PrefillMmParams& p, hipStream_t s);
int launch_prefill_mm_f32(const PrefillMmParams& p, hipStream_t s);
int launch_prefill_combine(const PrefillMmParams& p, hipStream_t s);

}  // namespace fd
