// Launches of differential attention for one 16-bit type.  diff_bf16.hip and
// diff_f16.hip include it after defining their debug-check flag words
// (PAL_DEBUG_FLAGS_DEFINE): the kernels of a type take minutes to compile.
#pragma once

#include "diff_decode.h"
#include "diff_tile.h"

namespace pal {
namespace {

template <int DT, int HD, int TPP, bool KV8>
hipError_t launch_diff_t(const DiffParams& p, hipStream_t stream) {
  const bool inline_plan = p.num_seqs <= kInlinePlanSeqs;
  if (!inline_plan) {
    if (p.q2seq)
      hipLaunchKernelGGL((diff_plan_kernel<HD, TPP>), dim3(1), dim3(kPlanThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((decode_plan_kernel<HD, TPP, kDiffSegmentCost>), dim3(1), dim3(kPlanThreads), 0, stream, p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  hipLaunchKernelGGL((diff_stream_kernel<DT, HD, TPP, KV8>),
                     dim3(static_cast<unsigned>(p.num_workers / kDiffWaves + (p.q2seq && inline_plan ? 1 : 0))), dim3(kDiffThreads), 0,
                     stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((diff_merge_kernel<DT, HD>), dim3(static_cast<unsigned>(p.num_workers), static_cast<unsigned>(p.hg_max)),
                     dim3(kDiffThreads), 0, stream, p);
  err = hipGetLastError();
  if (err != hipSuccess || !p.q2seq) return err;
  const int64_t items = (p.num_seqs / 2 + 1) * p.num_kv_heads * p.tile_chunks;  // at most
  const int64_t cus = p.num_workers / kDiffWaves;
  hipLaunchKernelGGL((diff_tile_kernel<DT, HD, TPP, KV8>), dim3(static_cast<unsigned>(items < cus ? items : cus)),
                     dim3(kPfThreads), sizeof(DiffTileLds<HD, KV8>), stream, p);
  return hipGetLastError();
}

template <int DT, int HD, bool KV8>
hipError_t launch_tpp(const DiffParams& p, int tpp, hipStream_t stream) {
  switch (tpp) {
    case 16: return launch_diff_t<DT, HD, 16, KV8>(p, stream);
    case 32: return launch_diff_t<DT, HD, 32, KV8>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

template <int DT>
hipError_t launch_hd(const DiffParams& p, int hd, int tpp, hipStream_t stream) {
  if (p.k_scales) {
    switch (hd) {
      case 64: return launch_tpp<DT, 64, true>(p, tpp, stream);
      case 128: return launch_tpp<DT, 128, true>(p, tpp, stream);
      default: return hipErrorInvalidValue;
    }
  }
  switch (hd) {
    case 32: return launch_tpp<DT, 32, false>(p, tpp, stream);
    case 64: return launch_tpp<DT, 64, false>(p, tpp, stream);
    case 96: return launch_tpp<DT, 96, false>(p, tpp, stream);
    case 128: return launch_tpp<DT, 128, false>(p, tpp, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace
}  // namespace pal
