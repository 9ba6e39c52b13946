// The matrix-core kernel of packed query tokens for fp16 (prefill_mm_kernel.h).
#include "prefill_mm_kernel.h"

namespace fd {
int launch_prefill_mm_f16(const PrefillMmParams& p, hipStream_t s) {
  return launch_prefill_mm<F16>(p, s);
}
}  // namespace fd
