// Differential attention of bfloat16 queries (kernels: diff_decode.h, diff_tile.h).
#include "pal_device.h"

namespace pal {

// flag word of this translation unit's debug checks (see pal_device.h)
PAL_DEBUG_FLAGS_DEFINE(diff_bf16_debug_flags)

}  // namespace pal

#include "diff_launch.h"

namespace pal {

hipError_t launch_diff_bf16(const DiffParams& p, int head_dim, int tokens_per_page, hipStream_t stream) {
  return launch_hd<kBF16>(p, head_dim, tokens_per_page, stream);
}

}  // namespace pal
