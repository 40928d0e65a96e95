// Differential attention over the paged cache for gfx950: the difference of two
// softmax maps with a learned weight, times a value of twice the head dim, and
// an RMS norm of the result.  The pools are those of ordinary attention: kv heads
// 2j and 2j + 1 of a page are two neighbouring blocks, [HD/x][TPP][x] keys and
// [HD][TPP] values, so the pair's value is one [2 HD][TPP] block.
//
// Decode rows (every row of the decode entry, the rows alone in their run of a
// mixed batch) are streamed in equal shares of the cache (diff_decode.h), the
// rows of chunks are MFMA tiles (diff_tile.h).  This file holds what is common to
// the query types.
#include "pal_device.h"

namespace pal {

hipError_t diff_resident_workers(int* workers) {
  int dev = 0, cus = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess) err = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  *workers = cus * 4;  // wavefronts: one workgroup of four per CU
  return err;
}

hipError_t launch_diff(const DiffParams& p, int dtype, int head_dim, int tokens_per_page, hipStream_t stream) {
  return dtype == kBF16 ? launch_diff_bf16(p, head_dim, tokens_per_page, stream)
                        : launch_diff_f16(p, head_dim, tokens_per_page, stream);
}

hipError_t diff_debug_flags(uint32_t* out, bool reset) {
  uint32_t other = 0;
  hipError_t err = diff_bf16_debug_flags(out, reset);
  if (err == hipSuccess) err = diff_f16_debug_flags(&other, reset);
  *out |= other;
  return err;
}

}  // namespace pal
