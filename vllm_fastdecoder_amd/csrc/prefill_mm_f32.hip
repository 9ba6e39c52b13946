// The matrix-core kernel of packed query tokens for fp32 (prefill_mm_kernel.h).
#include "prefill_mm_kernel.h"

namespace fd {
int launch_prefill_mm_f32(const PrefillMmParams& p, hipStream_t s) {
  return launch_prefill_mm<F32>(p, s);
}
}  // namespace fd
