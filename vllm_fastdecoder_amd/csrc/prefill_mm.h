// Attention of packed query tokens on the matrix cores: the
// kernel's plan and launcher, shared by prefill.hip (planning) and the
// translation units that instantiate it per type.
#pragma once

#include "prefill.h"

namespace fd {

// How a call is cut: A tasks take 32 query rows a wave of one row and kv
// head (row = token * group + head in the group), B tasks all of a row of at
// most kRowsB; each over parts of per_a / per_b steps of its keys.
struct PrefillPlan {
  int32_t tiles_a;  // A tiles at most, over all rows (0: no A tasks)
  int32_t rows_b;   // B tasks per kv head (n, or 0: none)
  int32_t waves;    // of a workgroup
  int32_t parts_a, per_a;  // parts at most, steps of each
  int32_t parts_b, per_b;
  size_t partial_bytes, counter_bytes;  // workspace: parts' results, arrival counters
};

constexpr int kRowsB = 64;
constexpr int kMostTileParts = 32;   // of an A tile's keys
constexpr int kMostRun = 16;         // keys whose place is looked up as one, at most
constexpr int kTableRoom = 4096;     // runs of a part at most (32 KiB of LDS; twice that if V's differ)
constexpr int kPrefillLds = 155 * 1024;    // of a workgroup, for its stages and tables
constexpr int kMaxPrefillCounters = 2048;  // 64-bit words of the caller's FD_DECODE_COUNTERS

struct PrefillMmParams {
  PrefillArgs a;
  PrefillPlan plan;
  int32_t G;
  float scale_log2;      // > 0
  uint32_t q_flip;       // sign bits to flip in a word of q (a negative scale)
  int32_t run_shift;     // keys whose place is looked up as one: 2^run_shift
  int64_t grid;
  int32_t stages;        // of K and V in LDS
  int32_t table_room;    // such runs of a part's keys at most
  bool alone;            // no more workgroups than CUs
  float* part_o;         // [parts][T * H][D]
  float2* part_ml;       // [parts][T * H]: running maximum (log2 domain) and sum
  uint64_t* counters;    // parts written, per (tile, kv head), counter_stride apart
  int32_t counter_stride;
  uint64_t launch;       // this launch's number, kLaunchBits up
};

PrefillPlan plan_prefill_mm(int32_t n, int32_t T, int32_t H, int32_t KVH, int32_t D, int32_t max_q,
                            int64_t max_k, int32_t BS, int32_t dt);
int launch_prefill_mm_f16(const PrefillMmParams& p, hipStream_t s);
int launch_prefill_mm_bf16(const PrefillMmParams& p, hipStream_t s);
int launch_prefill_mm_f32(const PrefillMmParams& p, hipStream_t s);

}  // namespace fd
