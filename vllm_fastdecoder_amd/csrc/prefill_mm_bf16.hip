// The matrix-core kernel of packed query tokens for bf16 (prefill_mm_kernel.h).
#include "prefill_mm_kernel.h"

namespace fd {
int launch_prefill_mm_bf16(const PrefillMmParams& p, hipStream_t s) {
  return launch_prefill_mm<BF16>(p, s);
}
}  // namespace fd
