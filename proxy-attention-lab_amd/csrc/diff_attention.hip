// Differential attention over the paged cache for gfx950: the difference of two
// softmax maps with a learned weight, times a value of twice the head dim, and
// an RMS norm of the result.  The pools are those of ordinary attention: kv heads
// 2j and 2j + 1 of a page are two neighbouring blocks, [HD/x][TPP][x] keys and
// [HD][TPP] values, so the pair's value is one [2 HD][TPP] block.
//
// Decode rows (every row of the decode entry, the rows alone in their run of a
// mixed batch) are streamed by diff_decode.h.  Rows of chunks: one wavefront per
// (row, output head): lane t scores key k0 + t of both maps, and then adds the
// block's values into the dims it owns, both maps' sums apart.
#include "pal_device.h"

namespace pal {

// flag word of this translation unit's debug checks (see pal_device.h)
PAL_DEBUG_FLAGS_DEFINE(diff_debug_flags)

}  // namespace pal

#include "diff_decode.h"

namespace pal {

namespace {

template <int DT, bool KV8>
__device__ __forceinline__ float pool_value(const void* pool, int64_t elem) {
  if constexpr (KV8) {
    const int code = static_cast<const uint8_t*>(pool)[elem];
    return __builtin_amdgcn_cvt_pk_f32_fp8(code, false)[0];
  } else {
    return Dt<DT>::to_f32(static_cast<const uint16_t*>(pool)[elem]);
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) v += shfl_xor(v, off);
  return v;
}

template <int DT, int HD, bool KV8>
__global__ __launch_bounds__(kWave) void diff_rows_kernel(const DiffParams p, int tpp) {
  constexpr int kOwn = 2 * HD / kWave;  // dims lane + 64 j
  constexpr int X = KV8 ? 16 : 8;       // dims of a key stripe
  __shared__ float q_lds[2 * HD];
  __shared__ float p_lds[2][kWave];
  __shared__ int64_t page_lds[kWave];
  const int lane = threadIdx.x;
  const int heads = p.num_q_heads / 2;
  const int64_t row = blockIdx.x / heads;
  const int head = static_cast<int>(blockIdx.x % heads);
  const int pair = head / p.group;
  int64_t seq = row, len = 0;
  if (p.q2seq) {
    const uint32_t sq = p.q2seq[row];
    if ((row == 0 || p.q2seq[row - 1] != sq) && (row + 1 == p.num_seqs || p.q2seq[row + 1] != sq)) return;  // a lone row
    seq = sq < p.num_pt_rows ? sq : 0;
    if (sq < p.num_pt_rows) len = min(p.seq_lens[sq], p.q_offset[row]);
  } else {
    len = p.seq_lens[row];
  }
  const int64_t max_tokens = p.page_table_width * tpp;
  PAL_DEBUG_FLAG(len > max_tokens, kDebugLength);
  len = len < 0 ? 0 : (len > max_tokens ? max_tokens : len);
  for (int d = lane; d < 2 * HD; d += kWave)  // q1, then q2
    q_lds[d] = Dt<DT>::to_f32(p.q[(row * p.num_q_heads + 2 * head) * HD + d]);
  __syncthreads();
  const int64_t block = static_cast<int64_t>(HD) * tpp;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][kOwn];
#pragma unroll
  for (int j = 0; j < kOwn; ++j) o[0][j] = o[1][j] = 0.f;
  for (int64_t k0 = 0; k0 < len; k0 += kWave) {
    const int64_t tok = k0 + lane;
    const int slot = static_cast<int>(tok % tpp);
    int64_t page = -1;  // < 0: not a key
    if (tok < len) {
      const uint32_t id = p.page_table[seq * p.page_table_width + tok / tpp];
      PAL_DEBUG_FLAG(id >= p.num_pages, kDebugPageId);
      if (id < p.num_pages) page = id;
    }
    page_lds[lane] = page;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      float s = -INFINITY;
      if (page >= 0) {
        const int64_t base = (page * 2 * p.num_kv_heads + 2 * pair + a) * block;
        float dot = 0.f;
        for (int d = 0; d < HD; ++d)
          dot += q_lds[a * HD + d] * pool_value<DT, KV8>(p.k_pool, base + (d / X * tpp + slot) * X + d % X);
        if constexpr (KV8) dot *= p.k_scales[page * 2 * p.num_kv_heads + 2 * pair + a];
        s = dot * p.scale_log2;
      }
      float top = fmaxf(m[a], s);
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) top = fmaxf(top, shfl_xor(top, off));
      const float ref = top == -INFINITY ? 0.f : top;
      const float alpha = __builtin_amdgcn_exp2f(m[a] - ref);
      const float e = __builtin_amdgcn_exp2f(s - ref);
      l[a] = l[a] * alpha + wave_sum(e);
#pragma unroll
      for (int j = 0; j < kOwn; ++j) o[a][j] *= alpha;
      m[a] = top;
      p_lds[a][lane] = e;
    }
    __syncthreads();
    const int n = static_cast<int>(min(static_cast<int64_t>(kWave), len - k0));
    for (int t = 0; t < n; ++t) {
      const int64_t pg = page_lds[t];
      if (pg < 0) continue;
      const int sl = static_cast<int>((k0 + t) % tpp);
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        const int d = lane + kWave * j;
        float v = pool_value<DT, KV8>(p.v_pool, (pg * 2 * p.num_kv_heads + 2 * pair) * block + static_cast<int64_t>(d) * tpp + sl);
        if constexpr (KV8) v *= p.v_scales[pg * 2 * p.num_kv_heads + 2 * pair + d / HD];
        o[0][j] += p_lds[0][t] * v;
        o[1][j] += p_lds[1][t] * v;
      }
    }
    __syncthreads();
  }
  const float i1 = l[0] > 0.f ? 1.f / l[0] : 0.f;
  const float i2 = l[1] > 0.f ? p.lambdas[head] / l[1] : 0.f;
  float x[kOwn], ss = 0.f;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    x[j] = o[0][j] * i1 - o[1][j] * i2;
    ss += x[j] * x[j];
  }
  float f = p.out_scale;
  if (p.norm_weight) f /= sqrtf(wave_sum(ss) / (2 * HD) + p.norm_eps);
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const int d = lane + kWave * j;
    float y = x[j] * f;
    if (p.norm_weight) y *= p.norm_weight[d];
    p.out[(row * heads + head) * 2 * HD + d] = Dt<DT>::from_f32(len > 0 ? y : 0.f);
  }
}

template <int DT, int HD, int TPP, bool KV8>
hipError_t launch_diff_t(const DiffParams& p, hipStream_t stream) {
  if (p.num_seqs > kInlinePlanSeqs) {
    hipLaunchKernelGGL((decode_plan_kernel<HD, TPP>), dim3(1), dim3(kPlanThreads), 0, stream, p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  hipLaunchKernelGGL((diff_stream_kernel<DT, HD, TPP, KV8>), dim3(static_cast<unsigned>(p.num_workers / kDiffWaves)),
                     dim3(kDiffThreads), 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((diff_merge_kernel<DT, HD>), dim3(static_cast<unsigned>(p.num_workers), static_cast<unsigned>(p.hg_max)),
                     dim3(kDiffThreads), 0, stream, p);
  err = hipGetLastError();
  if (err != hipSuccess || !p.q2seq) return err;
  const int64_t groups = p.num_seqs * (p.num_q_heads / 2);
  if (groups > 0x7fffffffLL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((diff_rows_kernel<DT, HD, KV8>), dim3(static_cast<unsigned>(groups)), dim3(kWave), 0, stream, p, TPP);
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

hipError_t diff_resident_workers(int* workers) {
  int dev = 0, cus = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess) err = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  *workers = cus * kDiffWaves;  // one workgroup per CU
  return err;
}

hipError_t launch_diff(const DiffParams& p, int dtype, int head_dim, int tokens_per_page, hipStream_t stream) {
  if (dtype == kBF16) return launch_hd<kBF16>(p, head_dim, tokens_per_page, stream);
  return launch_hd<kF16>(p, head_dim, tokens_per_page, stream);
}

}  // namespace pal
