// What a decode call's work list is made of, shared by the decode kernels and
// those of differential attention: the items (query rows with their keys), the
// cut of the list of 16-token blocks into virtual workers, the scan of the items'
// blocks for large batches, and lookups in it.  A translation unit includes it after defining its
// debug-check flag word (PAL_DEBUG_FLAGS_DEFINE).
#pragma once

#include "pal_device.h"

namespace pal {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kInlinePlanSeqs = 1024;  // largest batch scanned into LDS by each workgroup

struct Item {
  int64_t row;  // query / output row
  int64_t seq;  // page-table row
  int64_t len;  // visible keys, clamped to [0, W * TPP]
  bool skip;    // row mode: a row of a multi-row run (not ours to write)
};

__device__ __forceinline__ Item item_at(const DecodeParams& p, int64_t i, int tpp) {
  Item it;
  int64_t len;
  it.row = i;
  it.skip = false;
  if (p.q2seq) {
    const uint32_t sq = p.q2seq[i];
    it.skip = (i > 0 && p.q2seq[i - 1] == sq) || (i + 1 < p.num_seqs && p.q2seq[i + 1] == sq);
    if (sq < p.num_pt_rows && !it.skip) {
      it.seq = sq;
      len = p.seq_lens[sq];
      const int64_t off = p.q_offset[i];
      len = off < len ? off : len;
    } else {  // no such sequence, or a prefill row: nothing to attend to here
      it.seq = 0;
      len = 0;
    }
  } else {
    it.seq = i;
    len = p.seq_lens[i];
  }
  const int64_t max_tokens = p.page_table_width * tpp;
  PAL_DEBUG_FLAG(len > max_tokens, kDebugLength);
  it.len = len < 0 ? 0 : (len > max_tokens ? max_tokens : len);
  return it;
}

// The fixed cut of the global block list into virtual workers.
// Equal shares: [0, T) split evenly over nws = min(resident workers, T)
// virtual workers (none empty).  Fixed chunks: nc chunks of `chunk` blocks,
// virtual ids nws + k with nws = 0.  (A dynamically claimed tail of chunks
// after static shares measured much slower: each claimed range restarts the
// load pipeline and writes its own partials.)
struct Sched {
  int64_t total;  // T: blocks of all segments
  int64_t ts;     // static region [0, ts), split evenly over nws workers
  int64_t nws;    // static virtual workers
  int64_t chunk;  // blocks per chunk
  int64_t nc;     // chunks covering [ts, total); virtual ids nws .. nws + nc - 1
};

__device__ __forceinline__ Sched make_sched(int64_t total, int64_t nw, int tokens_per_worker) {
  Sched sc;
  sc.total = total;
  if (tokens_per_worker <= 0) {  // equal shares: no division on the start-up path
    sc.ts = total;
    sc.chunk = 1;
    sc.nws = total < nw ? total : nw;
    sc.nc = 0;
    return sc;
  }
  // fixed-size chunks (the reference's CHUNK_SIZE mode)
  sc.ts = 0;
  sc.chunk = tokens_per_worker / 16 > 0 ? tokens_per_worker / 16 : 1;
  sc.nws = 0;
  sc.nc = (total + sc.chunk - 1) / sc.chunk;
  return sc;
}

// First global block of virtual worker v (v in [0, nws + nc]); every virtual
// worker owns at least one block.
__device__ __forceinline__ int64_t vstart(const Sched& sc, int64_t v) {
  if (v <= sc.nws) return sc.nws > 0 ? (v * sc.ts) / sc.nws : 0;
  const int64_t b = sc.ts + (v - sc.nws) * sc.chunk;
  return b < sc.total ? b : sc.total;
}

// Virtual worker whose range holds global block b.
__device__ __forceinline__ int64_t vworker_of(const Sched& sc, int64_t b) {
  if (b < sc.ts) return ((b + 1) * sc.nws + sc.ts - 1) / sc.ts - 1;
  return sc.nws + (b - sc.ts) / sc.chunk;
}

// Zeros for every head of an empty item (no visible key).  Run by the
// planner's thread that finds the item; such items are rare.
template <int HD>
__device__ __forceinline__ void zero_item_output(const DecodeParams& p, int64_t row) {
  u32x2* o = reinterpret_cast<u32x2*>(p.out + row * p.num_q_heads * HD);  // out is 8-byte aligned
  const int64_t n = static_cast<int64_t>(p.num_q_heads) * HD / 4;
  for (int64_t i = 0; i < n; ++i) o[i] = u32x2{0u, 0u};
}

// Sequence holding global block b: the largest s with cum[s] <= b.
__device__ __forceinline__ int64_t locate_seq(const int64_t* cum, int64_t num_seqs, int64_t b) {
  int64_t lo = 0, hi = num_seqs - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (cum[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Scan for batches larger than kInlinePlanSeqs: cum[s] = first global block of
// sequence s (all of its segments), cum[S] = hdr[0] = T.  Each thread takes
// kPlanPer consecutive items per pass, so their length loads go out together;
// it also writes the zeros of an empty item.
constexpr int kPlanPer = 16;

template <int HD, int TPP, int kSegmentCost = 0>
__global__ __launch_bounds__(kPlanThreads) void decode_plan_kernel(const DecodeParams p) {
  __shared__ int64_t wave_sums[kPlanThreads / kWave];
  __shared__ int64_t carry_sh;
  const int64_t segs = static_cast<int64_t>(p.num_kv_heads) * p.head_chunks;
  const int tid = threadIdx.x;
  int64_t carry = 0;
  const int64_t n = p.num_seqs;
  for (int64_t base = 0; base < n; base += static_cast<int64_t>(kPlanThreads) * kPlanPer) {
    int64_t vals[kPlanPer];
    int64_t tsum = 0;
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) {
      const int64_t s = base + static_cast<int64_t>(tid) * kPlanPer + k;
      vals[k] = 0;
      if (s < n) {
        const Item it = item_at(p, s, TPP);
        vals[k] = it.len > 0 ? (((it.len + 15) >> 4) + kSegmentCost) * segs : 0;
        if (it.len == 0 && !it.skip) zero_item_output<HD>(p, it.row);
      }
      tsum += vals[k];
    }
    const int64_t inc = block_inclusive_scan<kPlanThreads>(tsum, wave_sums);
    int64_t c = carry + inc - tsum;
#pragma unroll
    for (int k = 0; k < kPlanPer; ++k) {
      const int64_t s = base + static_cast<int64_t>(tid) * kPlanPer + k;
      if (s < n) p.cum[s] = c;
      c += vals[k];
    }
    if (tid == kPlanThreads - 1) carry_sh = inc;
    __syncthreads();
    carry += carry_sh;
    __syncthreads();
  }
  if (tid == 0) {
    p.cum[n] = carry;
    p.hdr[0] = carry;
  }
}

}  // namespace
}  // namespace pal
