// Differential attention of query tiles (the rows of chunks) over the paged
// cache on gfx950 MFMA: the device code of a tile, and of the walk over a batch's
// tiles.
//
// For every row and output head, in one pass over the keys with running maxima
// and lazy rescaling (the formulas are in diff_decode.h): S_m^T = K_m Q_m^T and
// O_m^T += V^T P_m^T for the two maps m, the value V of 2 HD dims shared.
//
// Design (MI355X):
//  * One workgroup (4 wavefronts, one per SIMD) has a CU to itself and owns 128
//    "M-rows": consecutive query tokens of one sequence times the output heads
//    of a kv pair (up to 16 of them).  A wavefront holds 32 M-rows with BOTH maps
//    of each: an operand of V read from LDS feeds two MFMAs, a lane holds both
//    maps of its rows, so the difference, the norm and the output never cross
//    lanes but for one exchange of halves.  (One map per wavefront would read
//    24 KiB of LDS per 24 MFMAs and wavefront, all of the LDS' rate; this reads
//    32 KiB per 48.)
//  * Registers: the two maps' O is 2 x 32 x 2 HD fp32, half of the register file
//    at HD 128: 16 accumulators in v128.. and a128.., named by the MFMA
//    instructions (the compiler keeps to the registers below, as in
//    prefill_tile.h); below them the queries (64), the scores of this step and
//    the next (64), the probabilities and the operands in flight (about 44).
//  * Staging as in prefill_tile.h: per 32-key step K and V reach LDS by
//    direct-to-LDS copies, three to four steps ahead, four buffers each, one
//    barrier per step; the pair's two (page, kv head) blocks are neighbours, so
//    they are copied as one block of 2 HD dims.  Steps with an invalid page id
//    take a synchronous register path.
//  * Schedule of a step: QK MFMAs of the next step beside the exponentials of the
//    first 16 keys; PV MFMAs of the first 16 keys beside
//    the exponentials of the other 16; PV MFMAs of those beside the next step's
//    exponents and maxima.  So the 32 exponentials of a row pair (16 cycles
//    each) spread over all 48 MFMAs.
//  * fp8 pages are copied as codes and converted in the operand reads (exact).
//    Key scales go on the scores; value scales on the probabilities, which
//    are packed once for either half of the value.  With fp16 products the
//    power of two of a value scale goes into the conversion of the codes
//    instead, so that a small scale cannot push probabilities below fp16's range.
//  * Tiles are claimed from 8 counters (one for the workgroups of each XCD, the
//    others in turn when it is empty), which the stream kernel before clears.
//
// Measured (HD 128, bf16, 32 query heads on 4 kv pairs): 1.22 us a step, 1,317
// TFLOP/s, where a large matrix product reaches 1,384 on the same card.  A tile's
// start and end take about 14 us more (limits and page ids 6, first copies and
// scores 4, difference, norm and store 6 with the loop's last step beside it): 8
// chunks of 512-2,048 rows on 0-2,048 cached keys, 1,308 tiles, 400 us.  Over fp8
// pages the vector pipe bounds a step: 128 conversions and 64 scalings of
// probabilities beside the 48 products.
#pragma once

#include "diff_decode.h"
#include "prefill_tile.h"

namespace pal {
namespace {

constexpr int kDiffMRows = 128;  // M-rows of a tile
// Iteration st copies K of step st + kDiffLeadK (K operands of step st + 1 are
// still read in its first part, so that buffer may not be overwritten) and V of
// step st + kDiffLeadV; kLeadK and kLeadV of pid_window.h bound them.
constexpr int kDiffLeadK = 4, kDiffLeadV = 3;
static_assert(kDiffLeadK <= kLeadK && kDiffLeadV <= kLeadV && kDiffLeadK == kNBuf && kDiffLeadV == kNBuf - 1, "staging order");
constexpr int kDiffAcc = 128;    // first accumulator register, of either file
// (Two wavefronts per SIMD at most and LDS allocated at launch: where the
// compiler sees that only one fits, it takes 129 registers of either file at
// least.)
#define PAL_DIFF_TILE_KERNEL __attribute__((amdgpu_waves_per_eu(1, 2), amdgpu_num_vgpr(128)))

// accumulator I (0 .. 15): v[128 + 16 I ..] up to 7, a[128 + 16 (I - 8) ..] from 8 on
#define PAL_DIFF_MMA(type, file, acls)                                                                    \
  asm volatile("v_mfma_f32_32x32x16_" type " " file "[%2:%3], %0, %1, " file "[%2:%3]" ::acls(a), "v"(b), \
               "n"(kDiffAcc + 16 * (I & 7)), "n"(kDiffAcc + 16 * (I & 7) + 15))
#define PAL_DIFF_MMA_OF(type, acls)                     \
  do {                                                  \
    if constexpr (I < 8) PAL_DIFF_MMA(type, "v", acls); \
    else PAL_DIFF_MMA(type, "a", acls);                 \
  } while (0)
template <int DT, bool kAgprA, int I>
__device__ __forceinline__ void diff_mma(u32x4 a, u32x4 b) {
  if constexpr (DT == kBF16) {
    if constexpr (kAgprA) PAL_DIFF_MMA_OF("bf16", "a");
    else PAL_DIFF_MMA_OF("bf16", "v");
  } else {
    if constexpr (kAgprA) PAL_DIFF_MMA_OF("f16", "a");
    else PAL_DIFF_MMA_OF("f16", "v");
  }
}
#undef PAL_DIFF_MMA_OF
#undef PAL_DIFF_MMA
// s (+)= A B, 32x32x16, with B (a query operand) in AGPRs, where the compiler is to
// keep it: as a builtin's operand it was copied to VGPRs for each product.  The
// compiler does not see that s is an MFMA's result: whoever reads it stands 18
// wait states or more behind (acc_settle, or the PV MFMAs between).
#define PAL_DIFF_QK(type, acls)                                                                                     \
  do {                                                                                                              \
    if constexpr (kFirst) asm volatile("v_mfma_f32_32x32x16_" type " %0, %1, %2, 0" : "=&v"(s) : acls(a), "a"(b));  \
    else asm volatile("v_mfma_f32_32x32x16_" type " %0, %1, %2, %0" : "+v"(s) : acls(a), "a"(b));                   \
  } while (0)
template <int DT, bool kAgprA, bool kFirst>
__device__ __forceinline__ void diff_qk(f32x16& s, u32x4 a, u32x4 b) {
  if constexpr (DT == kBF16) {
    if constexpr (kAgprA) PAL_DIFF_QK("bf16", "a");
    else PAL_DIFF_QK("bf16", "v");
  } else {
    if constexpr (kAgprA) PAL_DIFF_QK("f16", "a");
    else PAL_DIFF_QK("f16", "v");
  }
}
#undef PAL_DIFF_QK
// element X (0 .. 255) of the accumulators
template <int X>
__device__ __forceinline__ float diff_acc_get() {
  float v;
  if constexpr (X < 128) asm volatile("v_mov_b32 %0, v[%1]" : "=v"(v) : "n"(kDiffAcc + X));
  else asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(v) : "n"(kDiffAcc + X - 128));
  return v;
}
// element X times f
template <int X>
__device__ __forceinline__ float diff_acc_mul(float f) {
  if constexpr (X < 128) {
    float v;
    asm volatile("v_mul_f32 %0, v[%1], %2" : "=v"(v) : "n"(kDiffAcc + X), "v"(f));
    return v;
  } else {
    return diff_acc_get<X>() * f;
  }
}
// element X (of the VGPRs) = itself times f plus t; ss += its square
template <int X>
__device__ __forceinline__ void diff_acc_join(float f, float t, float& ss) {
  static_assert(X < 128, "an accumulator in VGPRs");
  asm volatile("v_fma_f32 v[%1], v[%1], %2, %3\n\tv_fma_f32 %0, v[%1], v[%1], %0"
               : "+v"(ss)
               : "n"(kDiffAcc + X), "v"(f), "v"(t));
}
template <int X>
__device__ __forceinline__ void diff_acc_put(float v) {
  if constexpr (X < 128) asm volatile("v_mov_b32 v[%1], %0" ::"v"(v), "n"(kDiffAcc + X));
  else asm volatile("v_accvgpr_write_b32 a[%1], %0" ::"v"(v), "n"(kDiffAcc + X - 128));
}

// The kernel's parameters, read again from its argument segment: a place outside
// the step loop (set-up, slow paths, output) takes them from here, and a tile's
// coordinates from LDS, so that they hold no scalar registers through the loop.
// (For scalars that it spills the compiler takes a vector register past its
// limit, one of the accumulators'.)
typedef const __attribute__((address_space(4))) DiffParams DiffArgs;
__device__ __forceinline__ DiffArgs* diff_args() {
  DiffArgs* a = (DiffArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

// The lane, computed here and now: what is derived from the kernel's thread index
// the compiler computes once, before all tiles, and spills, and reading it back
// from scratch memory waits for every copy and store in flight (the output of a
// tile took 9.3 us of that).
__device__ __forceinline__ int lane_now() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
  return l;
}

// Steps of K (and of V): the 16-byte items of the pair's block
template <int HD, bool KV8>
struct DiffGeo {
  static constexpr int VD = 2 * HD;
  static constexpr int kItems = (KV8 ? 2 : 4) * VD;
  static constexpr int kCopies = (kItems + kPfThreads - 1) / kPfThreads;  // per thread, per K (or V)
};

// LDS of a tile workgroup.
template <int HD, bool KV8>
struct DiffTileLds {
  __attribute__((aligned(16))) uint16_t k[kNBuf * DiffGeo<HD, KV8>::kItems * 8];
  __attribute__((aligned(16))) uint16_t v[kNBuf * DiffGeo<HD, KV8>::kItems * 8];
  __attribute__((aligned(16))) uint16_t junk[kWave * 8];  // target of padding copies
  uint32_t pid[2 * kPidChunk];
  float scl[KV8 ? 8 * kPidChunk : 1];  // fp8: scales of each staged page id, [K1, K2, V1, V2][slot]
  int lim[kDiffMRows + 2 * kPfWaves + 1];
  uint64_t other[kDiffMRows / kWave];  // rows of another sequence than the tile's
  uint32_t next[4];  // the next item, its claim queue, and its tile's entry in the list
  int tile[8];  // the tile: first row, rows, kv pair, first head, heads, claim queue
  float lam[16];  // lambdas of the tile's heads
  __attribute__((aligned(16))) float weight[2 * HD];  // what a row is scaled with behind its norm
};

// Entry in the list of an item's tile: {first row, sequence}.
__device__ __forceinline__ const uint32_t* diff_entry(DiffArgs* p, unsigned item) {
  const unsigned index = item / (static_cast<unsigned>(p->num_kv_heads) * p->tile_chunks);
  return p->tiles + 2 * (p->hdr[3] ? index : static_cast<unsigned>(p->hdr[2]) - 1 - index);
}

// Item of claim n in queue q of a grid of nb workgroups: queue q has items q, q + 8,
// ..., whose first ceil((nb - q) / 8) are taken by place.
__device__ __forceinline__ unsigned diff_item_of(uint32_t q, uint32_t n, unsigned nb) {
  return q + kDiffQueues * (n + (nb + kDiffQueues - 1 - q) / kDiffQueues);
}

// Item `item`, head group item % G (G = kv pairs x head chunks) of the tile of
// sequence seq_u that begins at row row0.  Claims the next item behind its last
// step (while the norm is made; a claim at the tile's start would hand the last
// items to the workgroups that began first, which have the longest).
template <int DT, int HD, int TPP, bool KV8>
__device__ __forceinline__ void diff_tile(unsigned item, uint32_t queue, int row0, uint32_t seq_u,
                                          DiffTileLds<HD, KV8>& L) {
  constexpr int VD = 2 * HD;
  constexpr int KS = HD / 16;  // QK k-steps of a map; also row tiles of 32 value dims
  constexpr int NQ = 2 * KS;   // QK MFMAs of a step (and PV operands, two MFMAs each)
  constexpr int NI = DiffGeo<HD, KV8>::kItems;
  constexpr int NC = DiffGeo<HD, KV8>::kCopies;
  constexpr bool F8 = KV8;
  constexpr bool kSplitScale = F8 && DT == kF16;  // value scales: power of two on the codes, the rest on P
  using IM = ItemMap<VD, TPP>;
  auto k_lds = [&](int j) { return L.k + (j & (kNBuf - 1)) * NI * 8; };  // step j's buffer
  auto v_lds = [&](int j) { return L.v + (j & (kNBuf - 1)) * NI * 8; };
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };

  DiffArgs* args = diff_args();
  const unsigned G = static_cast<unsigned>(args->num_kv_heads) * args->tile_chunks;
  const unsigned grp = item % G;
  const int tile_heads = args->tile_heads;
  const int pair = static_cast<int>(grp / args->tile_chunks);
  const int h0 = static_cast<int>(grp % args->tile_chunks) * tile_heads;
  const int hg = min(tile_heads, args->group - h0);
  const bool seq_ok = seq_u < args->num_pt_rows;  // a row naming no sequence attends to nothing
  const int64_t s = seq_ok ? seq_u : 0;
  const int qt = args->tile_rows;  // tokens per tile
  const int lane = lane_now();
  const int w = wave_id();
  const int tid = w * kWave + lane;
  const int col = lane & 31;  // this lane's M-row within the wavefront's
  const int half = lane >> 5;

  const int64_t max_tokens = args->page_table_width * TPP;
  int64_t slen = seq_ok ? args->seq_lens[s] : 0;
  PAL_DEBUG_FLAG(slen > max_tokens, kDebugLength);
  slen = slen < 0 ? 0 : (slen > max_tokens ? max_tokens : slen);

  // The loads that need only the tile's coordinates: its rows' sequences and key
  // limits, first page-table entries, queries.  (Rows past the tile's run are found
  // out below; they may be read as if they were the tile's.)
  constexpr int kBad = kDiffMRows + 2 * kPfWaves;  // L.lim word set when a staged page id is out of range
  const int64_t n_rows = args->num_seqs;
  const bool in = tid < qt && row0 + tid < n_rows;
  const uint32_t row_seq = in ? args->q2seq[row0 + tid] : ~seq_u;
  const int tok_off = in ? args->q_offset[row0 + tid] : 0;
  const uint32_t* pt0 = args->page_table + s * args->page_table_width;
  constexpr int kPidPre = kPidChunk / kPfThreads;
  uint32_t pid_pre[kPidPre];
#pragma unroll
  for (int j = 0; j < kPidPre; ++j) {
    const int e = tid + j * kPfThreads;
    pid_pre[j] = e < args->page_table_width ? pt0[e] : 0u;
  }
  const int m_row = w * 32 + col;
  const int my_t = static_cast<int>((static_cast<uint32_t>(m_row) * args->tile_magic) >> 16);  // m_row / tile_heads
  const int my_h = m_row - my_t * tile_heads;
  const bool may = my_t < qt && row0 + my_t < n_rows && my_h < hg;
  const int head = pair * args->group + h0 + (may ? my_h : 0);
  // Q^T operands of both maps: Q[M-row col][16 kk + 8 half .. +7] (an M-row past
  // the tile takes the first's; its result is not written); fp8 steps: k-step
  // 2j + e takes dims 16 (2j + half) + 8e .. +7, as the key items hold them
  u32x4 qv[2][KS];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint16_t* qp = args->q + (static_cast<int64_t>(row0 + (may ? my_t : 0)) * args->num_q_heads + 2 * head + r) * HD;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
      qv[r][kk] = *reinterpret_cast<const u32x4*>(qp + (F8 ? 32 * (kk / 2) + 16 * half + 8 * (kk % 2) : 16 * kk + 8 * half));
  }
  __syncthreads();  // the previous tile is done with every LDS array
  if (tid < 16) L.lam[tid] = args->lambdas[pair * args->group + h0 + (tid < hg ? tid : 0)];
  if (tid < VD) L.weight[tid] = args->out_scale * (args->norm_weight ? args->norm_weight[tid] : 1.f);
  if (w < kDiffMRows / kWave) {
    const uint64_t m = __ballot(row_seq != seq_u);
    if (lane == 0) L.other[w] = m;
  }
  __syncthreads();
  // rows of the tile: up to the first of another sequence (or the last of the call)
  int nrows = qt;
#pragma unroll
  for (int i = kDiffMRows / kWave - 1; i >= 0; --i) {
    const uint64_t m = (static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(L.other[i] >> 32)))) << 32) |
                       static_cast<uint32_t>(uniform(static_cast<int>(L.other[i])));
    if (m) nrows = min(qt, i * kWave + static_cast<int>(__builtin_ctzll(m)));
  }
  const bool row_ok = may && my_t < nrows;
  {
    const bool live = tid < nrows;
    int lim = 0;
    if (live) {
      const int64_t off = tok_off < 0 ? 0 : tok_off;
      lim = static_cast<int>(off < slen ? off : slen);
    }
    if (tid < kDiffMRows) L.lim[tid] = lim;
    const int mx = wave_max(lim);
    const int mn = -wave_max(live ? -lim : -(1 << 30));
    if (lane == 0) {
      L.lim[kDiffMRows + w] = mx;
      L.lim[kDiffMRows + kPfWaves + w] = mn;
    }
    if (tid == 0) {
      L.lim[kBad] = 0;
      L.tile[0] = row0;
      L.tile[1] = nrows;
      L.tile[2] = pair;
      L.tile[3] = h0;
      L.tile[4] = hg;
      L.tile[5] = static_cast<int>(queue);
    }
  }
  __syncthreads();
  int max_lim = 0, min_lim = 1 << 30;
#pragma unroll
  for (int i = 0; i < kPfWaves; ++i) {
    max_lim = max(max_lim, L.lim[kDiffMRows + i]);
    min_lim = min(min_lim, L.lim[kDiffMRows + kPfWaves + i]);
  }
  max_lim = __builtin_amdgcn_readfirstlane(max_lim);
  min_lim = __builtin_amdgcn_readfirstlane(min_lim);
  const int my_lim = row_ok ? L.lim[my_t] : 0;

  const int64_t pair_block = static_cast<int64_t>(VD) * TPP;  // elements of a pair's block
  const int64_t page_stride = pair_block * args->num_kv_heads;
  const int nsteps = (max_lim + kKeys - 1) / kKeys;
  const int n_pid = (max_lim + TPP - 1) / TPP;  // page-table entries the tile reads: never past the width

  // Page ids (and fp8 scales) live in LDS, two chunks of 512 entries, entry e in
  // slot e % 1024, so the only vector-memory traffic of the step loop is the
  // copies, whose count its waits rely on.
  auto stage_pid = [&](DiffArgs* a0, int e, uint32_t pg) {
    L.pid[pid_slot(e)] = pg;
    const bool ok = pg < a0->num_pages;
    if (!ok) L.lim[kBad] = 1;
    if constexpr (F8) {  // (0 for an invalid id: such a step's codes are zeros)
      const int64_t si = 2 * (static_cast<int64_t>(ok ? pg : 0) * a0->num_kv_heads + uniform(L.tile[2]));
#pragma unroll
      for (int a = 0; a < 4; ++a)
        L.scl[a * 2 * kPidChunk + pid_slot(e)] = ok ? (a < 2 ? a0->k_scales : a0->v_scales)[si + (a & 1)] : 0.f;
    }
  };
  auto stage_pids = [&](int chunk) {  // synchronous; callers hold a barrier after it
    DiffArgs* a = diff_args();
    const uint32_t* pt = a->page_table + s * a->page_table_width;
    for (int e = chunk * kPidChunk + w * kWave + lane_now(); e < min((chunk + 1) * kPidChunk, n_pid); e += kPfThreads)
      stage_pid(a, e, pt[e]);
  };

  // Items of a step (see prefill_tile.h; the pair's block as one of VD dims).
  constexpr bool kAllItems = NI % kPfThreads == 0;  // no wavefront has a padding copy
  __builtin_assume(w >= 0 && w < kPfWaves);
  const bool long_pages = page_stride * (F8 ? 1 : 2) > 0xFFFFFFFFll;  // copies take a page's stride as 32 bits
  const uint32_t valid_pages = args->num_pages > 0xFFFFFFFFll ? 0xFFFFFFFFu : static_cast<uint32_t>(args->num_pages);
  const uint32_t np32 = long_pages ? 0u : valid_pages;  // pages the copies take
  auto k8_item = [](int i, int& ph, int& c, int& key) {
    if (TPP == 16) {  // page-major; page 1's keys at positions XOR 12, so a 16-lane operand read spans all banks
      ph = i / VD;
      c = (i % VD) / 16;
      key = 16 * ph + ((i % 16) ^ (ph ? 12 : 0));
    } else {
      ph = 0;
      c = i / 32;
      key = kperm_f8(i % 32);
    }
  };
  auto v8_item = [](int i, int& ph, int& d, int& kb) {
    ph = TPP == 16 ? i / VD : 0;
    d = i % VD;
    kb = 16 * (i / VD);
  };
  auto wave_item = [&](int q) { return w * kWave + q * kPfThreads; };
  auto live_copy = [&](int q) { return kAllItems || wave_item(q) < NI; };
  const uint64_t k_pair = reinterpret_cast<uint64_t>(args->k_pool) + pair * pair_block * (F8 ? 1 : 2);
  const uint64_t v_pair = reinterpret_cast<uint64_t>(args->v_pool) + pair * pair_block * (F8 ? 1 : 2);
  const uint32_t page_bytes = static_cast<uint32_t>(page_stride * (F8 ? 1 : 2));
  // A wavefront's copy q moves items 64 (w + 4 q) ..: 1 KiB of LDS and, in a page,
  // the items of 64 lanes at a fixed pattern from a place that the wavefront and q
  // give, so that one address per page serves the copies in it.
  constexpr int kChunksPerPage = (TPP == 16 ? NI / 2 : NI) / kWave;
  auto copy_half = [&](int q) { return TPP == 16 ? (w + kPfWaves * q) / kChunksPerPage : 0; };  // page half
  // bytes from the lane's place in a page to copy q's (fp8 V items of 32-token
  // pages: rows of 32 bytes, the second 16 keys behind the first VD rows)
  auto k_rel = [&](int q) { return static_cast<uint32_t>((w + kPfWaves * q) % kChunksPerPage) * 1024u; };
  auto v_rel = [&](int q) {
    const int c = w + kPfWaves * q;
    if (F8 && TPP == 32) return static_cast<uint32_t>((c % (VD / kWave)) * 2048 + 16 * (c / (VD / kWave)));
    return static_cast<uint32_t>(c % kChunksPerPage) * 1024u;
  };
  // places of the lane's item in the wavefront's chunks (its pattern repeats every
  // 4 chunks; fp8 keys of page half 1 are at positions XOR 12)
  uint64_t k_lane, k_lane1 = 0, v_lane;
  if constexpr (F8) {
    k_lane = k_pair + static_cast<uint32_t>(TPP == 16 ? lane * 16 : ((lane / 32) * 32 + kperm_f8(lane % 32)) * 16);
    k_lane1 = k_pair + static_cast<uint32_t>((lane ^ 12) * 16);
    v_lane = v_pair + static_cast<uint32_t>(lane * TPP);
  } else {
    int d, key;
    k_lane = k_pair + 2u * static_cast<uint32_t>(IM::k_offset(lane));
    IM::v_item(w * kWave + lane, d, key);
    v_lane = v_pair + 2u * static_cast<uint32_t>((d - (TPP == 16 ? 32 : 16) * (w % kChunksPerPage)) * TPP + key % TPP);
  }
  auto copy = [](uint64_t addr, uint32_t lds) {  // (the s_nop is the wait state after the M0 write)
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(addr), "{m0}"(lds) : "memory");
  };
  auto copy_k = [&](int q, int j, uint32_t pg0, uint32_t pg1) {
    const bool ok = live_copy(q);
    const bool ph = ok && copy_half(q);
    copy((F8 && TPP == 16 && ph ? k_lane1 : k_lane) + static_cast<uint64_t>(ph ? pg1 : pg0) * page_bytes + (ok ? k_rel(q) : 0u),
         lds_addr(ok ? k_lds(j) + wave_item(q) * 8 : L.junk));
  };
  auto copy_v = [&](int q, int j, uint32_t pg0, uint32_t pg1) {
    const bool ok = live_copy(q);
    copy(v_lane + static_cast<uint64_t>(ok && copy_half(q) ? pg1 : pg0) * page_bytes + (ok ? v_rel(q) : 0u),
         lds_addr(ok ? v_lds(j) + wave_item(q) * 8 : L.junk));
  };
  // a step whose pages are valid is copied (the tile's last may end past max_lim:
  // fix_tail clears the values of keys no row sees)
  auto is_fast = [&](int j, uint32_t pg0, uint32_t pg1) { return j * kKeys < max_lim && pg0 < np32 && pg1 < np32; };
  // the register path: zeros for invalid pages and keys past max_lim; drains the
  // copies in flight, which keeps the counted waits safe
  auto slow_k = [&](int j, uint32_t pg0, uint32_t pg1) {
    uint16_t* kb = k_lds(j);
    DiffArgs* a = diff_args();
    const int64_t stride = pair_block * a->num_kv_heads * (F8 ? 1 : 2);  // bytes of a page
    const uint64_t from = reinterpret_cast<uint64_t>(a->k_pool) + uniform(L.tile[2]) * pair_block * (F8 ? 1 : 2);
    const int first = w * kWave + lane_now();
#pragma unroll 1
    for (int q = 0; q < NC; ++q) {
      const int i = first + q * kPfThreads;
      if (i >= NI) continue;
      int ph, c, key;
      if constexpr (F8) {
        k8_item(i, ph, c, key);
      } else {
        ph = IM::k_page_half(i);
        IM::k_item(i, c, key);
      }
      const uint32_t pg = ph ? pg1 : pg0;
      PAL_DEBUG_FLAG(pg >= a->num_pages && j * kKeys + key < max_lim, kDebugPageId);
      u32x4 val = {0u, 0u, 0u, 0u};
      if (pg < a->num_pages && j * kKeys + key < max_lim)
        val = *reinterpret_cast<const u32x4*>(from + pg * stride + (c * TPP + key % TPP) * 16);
      *reinterpret_cast<u32x4*>(kb + i * 8) = val;
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  };
  // of an item's keys (8 of 16 bits, 16 of 8), the first `valid`
  auto keep_keys = [](u32x4 val, int valid) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t keep = 0;
      if constexpr (F8) {
#pragma unroll
        for (int b = 0; b < 4; ++b) keep |= 4 * e + b < valid ? 0xFFu << (8 * b) : 0u;
      } else {
        keep = (2 * e < valid ? 0x0000FFFFu : 0u) | (2 * e + 1 < valid ? 0xFFFF0000u : 0u);
      }
      val[e] &= keep;
    }
    return val;
  };
  auto v_place = [&](int i, int& ph, int& d, int& key) {
    if constexpr (F8) {
      v8_item(i, ph, d, key);
    } else {
      ph = IM::k_page_half(i);
      IM::v_item(i, d, key);
    }
  };
  auto slow_v = [&](int j, uint32_t pg0, uint32_t pg1) {
    uint16_t* vb = v_lds(j);
    DiffArgs* a = diff_args();
    const int64_t stride = pair_block * a->num_kv_heads * (F8 ? 1 : 2);
    const uint64_t from = reinterpret_cast<uint64_t>(a->v_pool) + uniform(L.tile[2]) * pair_block * (F8 ? 1 : 2);
    const int first = w * kWave + lane_now();
#pragma unroll 1
    for (int q = 0; q < NC; ++q) {
      const int i = first + q * kPfThreads;
      if (i >= NI) continue;
      int ph, d, key;
      v_place(i, ph, d, key);
      const uint32_t pg = ph ? pg1 : pg0;
      const int valid = max_lim - (j * kKeys + key);
      u32x4 val = {0u, 0u, 0u, 0u};
      if (pg < a->num_pages && valid > 0)
        val = keep_keys(*reinterpret_cast<const u32x4*>(from + pg * stride + (d * TPP + key % TPP) * (F8 ? 1 : 2)), valid);
      *reinterpret_cast<u32x4*>(vb + i * 8) = val;
    }
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  };
  // Clears the values of keys past max_lim in the tile's last step j (a masked
  // probability of 0 times a NaN there would be NaN): each thread its own items,
  // once its copies have landed, before the barrier preceding the step's reads.
  auto fix_tail = [&](int j) {
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    compiler_fence();
    uint16_t* vb = v_lds(j);
    const int first = w * kWave + lane_now();
#pragma unroll 1
    for (int q = 0; q < NC; ++q) {
      const int i = first + q * kPfThreads;
      if (i >= NI) continue;
      int ph, d, key;
      v_place(i, ph, d, key);
      const int valid = max_lim - j * kKeys - key;
      if (valid < (F8 ? 16 : 8)) {
        u32x4* slot = reinterpret_cast<u32x4*>(vb + i * 8);
        *slot = keep_keys(*slot, valid);
      }
    }
  };
  const bool tail_partial = max_lim % kKeys != 0;
  auto read_pids = [&](int j) {  // the page ids of step j (LDS broadcast; TPP 32: one page)
    const int e = pid_slot(j * (kKeys / TPP));
    u32x2 v;
    if (TPP == 16) {
      v = *reinterpret_cast<const u32x2*>(L.pid + e);
    } else {
      v.x = L.pid[e];
      v.y = v.x;
    }
    return v;
  };
  // fp8: scale array a of the page of this lane's keys of step j (16 half .. +15);
  // 0 past the tile's last staged entry (0 x a stale scale could be NaN)
  auto read_scale = [&](int a, int j) {
    const int e = j * (kKeys / TPP) + (TPP == 16 ? half : 0);
    const float x = L.scl[a * 2 * kPidChunk + pid_slot(e)];
    return e < n_pid ? x : 0.f;
  };

  // minus the running max of this lane's M-row per map (log2 units); kNoMax until
  // the row's first score above -inf
  float mb[2] = {0.f, 0.f};
  float l_run[2] = {0.f, 0.f};  // this lane's share of the exp-sums
  asm volatile("" ::: "v255", "a255");  // the kernel allocates the accumulators' registers
  // K operand c = 2 kk + r: k-step kk of map r.  fp8: 8 codes of a 16-byte item
  // that holds k-steps kk and kk ^ 1
  using Op = std::conditional_t<F8, u32x2, u32x4>;
  auto read_k = [&](int j, int c) {
    const int r = c % 2, kk = c / 2;
    if constexpr (F8) {
      const int key = kperm_f8(col);
      const int st = r * (HD / 16) + 2 * (kk / 2) + half;
      const int slot = TPP == 16 ? (key / 16) * VD + st * 16 + ((key % 16) ^ (key >= 16 ? 12 : 0)) : st * 32 + col;
      return *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint8_t*>(k_lds(j)) + slot * 16 + 8 * (kk % 2));
    } else {
      return *reinterpret_cast<const u32x4*>(k_lds(j) + IM::k_slot(col, r * (HD / 8) + 2 * kk + half) * 8);
    }
  };
  // QK MFMA c of a step (fp8: the codes are exact in 16 bits, the key scale goes on
  // the scores; two instructions between a conversion and the MFMA that reads it)
  auto qk = [&](auto cc, f32x16(&sc)[2], Op v) {
    constexpr int c = decltype(cc)::value;
    if constexpr (F8) {
      u32x4 x = fp8x8_exact<DT>(v);
      asm volatile("s_nop 1" : "+v"(x));
      diff_qk<DT, false, (c < 2)>(sc[c % 2], x, qv[c % 2][c / 2]);
    } else {
      diff_qk<DT, true, (c < 2)>(sc[c % 2], v, qv[c % 2][c / 2]);
    }
  };
  // PV operand m: k-step m / KS, row tile m % KS (fp8: the lane's 16 keys of a row
  // are one item, 8 to a k-step)
  const int v_base[2] = {IM::v_slot(col, 8 * half), IM::v_slot(col, 16 + 8 * half)};
  auto read_v = [&](int j, int m) {
    if constexpr (F8)
      return *reinterpret_cast<const u32x2*>(reinterpret_cast<const uint8_t*>(v_lds(j)) +
                                             (half * VD + col + 32 * (m % KS)) * 16 + 8 * (m / KS));
    else
      return *reinterpret_cast<const u32x4*>(v_lds(j) + (v_base[m / KS] + (m % KS) * IM::kVRowTile) * 8);
  };
  // score register x is key 16 (x/8) + 8 half + 4 ((x/4)%2) + x%4 of the step (fp8: 16 half + x)
  auto place = [](int x) { return F8 ? x : 16 * (x >> 3) + 4 * ((x >> 2) & 1) + (x & 3); };
  // Register x of step j's scores is a key the row sees where place(x) is below
  // seen(j).of(x): keys below the row's limit, in a valid page.
  struct Seen {
    int lo, hi;  // registers 0 .. 7 and 8 .. 15 (fp8: the lane's keys are one page's)
    __device__ __forceinline__ int of(int x) const { return x < 8 ? lo : hi; }
  };
  auto seen = [&](int j) {
    const int lim = my_lim - j * kKeys - (F8 ? 16 : 8) * half;
    const u32x2 pg = read_pids(j);
    const bool ok0 = pg.x < valid_pages, ok1 = pg.y < valid_pages;
    if (F8) {
      const int l = (half ? ok1 : ok0) ? lim : -1;
      return Seen{l, l};
    }
    return Seen{ok0 ? lim : -1, ok1 ? lim : -1};
  };
  const float scale_log2 = args->scale_log2;
  auto score_scale = [&](int r, int j) { return F8 ? scale_log2 * read_scale(r, j) : scale_log2; };

  if (nsteps > 0) {
#pragma unroll
    for (int j = 0; j < kPidPre; ++j) {  // chunk 0, loaded above
      const int e = tid + j * kPfThreads;
      if (e < n_pid) stage_pid(args, e, pid_pre[j]);
    }
    if (n_pid > kPidChunk) stage_pids(1);
  }
  // the query loads are waited for here (the compiler would otherwise wait for them,
  // and so for the copies, inside the step loops)
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) asm volatile("" : "+a"(qv[r][kk]));
  __syncthreads();
  auto barrier = [&] {
    __builtin_amdgcn_s_waitcnt(kLgkmZero);
    __builtin_amdgcn_s_barrier();
    compiler_fence();
  };
  f32x16 e_cur[2];
  auto step_max = [&](bool masked, Seen vis, const f32x16& sv, float sc) {
    float bm = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x)
      if (!masked || place(x) < vis.of(x)) bm = fmaxf(bm, sv[x] * sc);
    return max_xor32(bm);
  };
  auto exponents = [&](int r, bool masked, Seen vis, const f32x16& sv, float sc) {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float v = fmaf(sv[x], sc, mb[r]);
      e_cur[r][x] = !masked || place(x) < vis.of(x) ? v : -INFINITY;
    }
  };
  // Operand reads of a step, in the order of their use: the rest of K (the first
  // kAhead operands are read in the step before), V, and the next K's first.  They
  // go out evenly, two to three MFMAs, 5 to 15 MFMAs ahead of their use: with all
  // of K read in the PV half and all of V in the QK half, the LDS would be
  // asked for its whole rate in the latter, and twice the registers hold
  // operands.
  constexpr int kAhead = HD == 128 ? (F8 ? 6 : 8) : (HD == 96 ? 8 : NQ);
  Op ka[NQ];
  const int paged_full = !long_pages ? max_lim / kKeys : 0;  // whole steps
  if (nsteps > 0) {
    auto pids = [&](int j, uint32_t& a, uint32_t& b) {
      const u32x2 v = read_pids(j);
      a = __builtin_amdgcn_readfirstlane(v.x);
      b = TPP == 16 ? __builtin_amdgcn_readfirstlane(v.y) : a;
    };
    // K 0, K 1, V 0, K 2, V 1, K 3, V 2
#pragma unroll 1
    for (int t = 0; t < 7; ++t) {
      const bool is_k = t == 0 || (t & 1);
      const int j = is_k ? (t + 1) / 2 : t / 2 - 1;
      if (j >= nsteps) continue;
      uint32_t pa, pb;
      pids(j, pa, pb);
      if (is_fast(j, pa, pb)) {
#pragma unroll
        for (int q = 0; q < NC; ++q) {
          if (is_k) copy_k(q, j, pa, pb);
          else copy_v(q, j, pa, pb);
        }
      } else if (is_k) {
        slow_k(j, pa, pb);
      } else {
        slow_v(j, pa, pb);
      }
    }
    static_for<2 * KS * 16>([](auto x) { diff_acc_put<decltype(x)::value>(0.f); });
    compiler_fence();
    if (nsteps >= 4)
      __builtin_amdgcn_s_waitcnt(vmcnt_only(5 * NC));  // K steps 0 and 1
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    if (nsteps == 1 && tail_partial) fix_tail(0);
    barrier();
    f32x16 s0[2];
#pragma unroll
    for (int c = 0; c < NQ; ++c) ka[c] = read_k(0, c);
    static_for<NQ>([&](auto cc) { qk(cc, s0, ka[decltype(cc)::value]); });
    acc_settle();
#pragma unroll
    for (int c = 0; c < kAhead; ++c) ka[c] = read_k(1, c);
    const Seen vis = seen(0);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float sc = score_scale(r, 0);
      const float bm = step_max(true, vis, s0[r], sc);
      mb[r] = bm == -INFINITY ? kNoMax : -bm;
      exponents(r, true, vis, s0[r], sc);
    }
  }

  // One iteration (memory and compute pipeline as in prefill_tile.h).  kFast: step
  // st + 1 needs no mask and the copied steps are whole and valid.  kLast: the
  // tile's last step.
  enum { kFast, kAny, kLast };
  auto step = [&](auto mode_c, int st) {
    constexpr int kMode = decltype(mode_c)::value;
    compiler_fence();
    // K of step st + 2 and V of step st have landed: all copies but V of st + 1, K of
    // st + 3 and V of st + 2, where there are those
    if (kMode == kFast || st + 3 < nsteps)
      __builtin_amdgcn_s_waitcnt(vmcnt_only(3 * NC));
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    barrier();
    const int jk = st + kDiffLeadK, jv = st + kDiffLeadV;
    const u32x2 pgk = read_pids(jk), pgv = read_pids(jv);  // (in bounds whether or not the steps exist)
    if (kMode == kAny && st + 2 == nsteps && tail_partial) fix_tail(st + 1);
    // written in issue order, chunk by chunk, with scheduling fences between
    sched_fence();
    float vsm[2] = {1.f, 1.f}, vse[2] = {1.f, 1.f};  // fp8: value scales of the halves, on P and on the codes
    if constexpr (F8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = read_scale(2 + h, st);
        vsm[h] = x;
        if constexpr (kSplitScale) {
          const uint32_t b = __float_as_uint(x);
          const bool special = (b & 0x7F800000u) == 0x7F800000u;
          vsm[h] = special ? x : __uint_as_float((b & 0x807FFFFFu) | 0x3F800000u);
          vse[h] = special ? 1.f : __uint_as_float(b & 0x7F800000u);
        }
      }
    }
    f32x16 s_next[2];
    Op va[NQ];
    constexpr int NP = F8 ? 2 : 1;  // packed probabilities: one per half of the value over fp8 pages
    u32x4 pp[2][2][NP];             // [map][k-step]
    // probability pair q: k-step q / 8, map (q / 4) % 2, pair q % 4 of the lane's 8 keys
    auto pair_exp = [&](int q) {
      const int r = (q / 4) % 2, x = 8 * (q / 8) + 2 * (q % 4);
      e_cur[r][x] = __builtin_amdgcn_exp2f(e_cur[r][x]);
      e_cur[r][x + 1] = __builtin_amdgcn_exp2f(e_cur[r][x + 1]);
    };
    auto pair_pack = [&](int q) {
      const int r = (q / 4) % 2, ks = q / 8, i = q % 4, x = 8 * ks + 2 * i;
      const float p0 = e_cur[r][x], p1 = e_cur[r][x + 1];
      l_run[r] += p0;
      l_run[r] += p1;
#pragma unroll
      for (int h = 0; h < NP; ++h) {
        // held here: code motion would sink the conversion to the MFMA that reads
        // it, which (as inline assembly) must stand two instructions behind it
        if constexpr (F8) {
          uint32_t w = Dt<DT>::pack2(p0 * vsm[h], p1 * vsm[h]);
          asm volatile("" : "+v"(w));
          pp[r][ks][h][i] = w;
        } else {
          pp[r][ks][h][i] = Dt<DT>::pack2(p0, p1);
          if (i == 3) asm volatile("" : "+v"(pp[r][ks][h]));
        }
      }
    };
    // the operand reads that go out with MFMA n of the step's 3 NQ
    auto reads_at = [&](auto nc) {
      constexpr int n = decltype(nc)::value;
      static_for<2>([&](auto ii) {
        constexpr int i = 2 * (n / 3) + decltype(ii)::value;  // read i goes out with MFMA 3 i / 2
        if constexpr (3 * i / 2 == n) {
          constexpr int kRest = NQ - kAhead;
          if constexpr (i < kRest) {
            if constexpr (kMode != kLast) ka[kAhead + i] = read_k(st + 1, kAhead + i);
          } else if constexpr (i < kRest + NQ) {
            va[i - kRest] = read_v(st, i - kRest);
          } else {
            if constexpr (kMode != kLast) ka[i - kRest - NQ] = read_k(st + 2, i - kRest - NQ);
          }
        }
      });
    };
    auto convert_k = [&](auto c) {  // fp8: an operand from its codes
      if constexpr (F8) return fp8x8_exact<DT>(c);
      else return c;
    };
    auto convert_v = [&](int m, auto c) {  // fp8: operand m from its codes
      if constexpr (kSplitScale) {
        const float e = vse[(m % KS) / (KS / 2)];
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f16x2 v = i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i / 2], e, true)
                                : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i / 2], e, false);
          r[i] = __builtin_bit_cast(uint32_t, v);
        }
        return r;
      } else {
        return convert_k(c);
      }
    };
    // fp8: operands are converted a chunk ahead of their MFMA, before the chunk's
    // other work: an MFMA stands two wait states or more behind a conversion (with
    // conversions right before their MFMA and the waits filled with s_nop, 4 chunks
    // of 256-1,024 rows on 0-4,096 keys of HD 128 took 235 us, now 226)
    u32x4 op[2];
    auto converted = [&](int i) {
      asm volatile("" : "+v"(op[i]));
      sched_fence();
    };
    auto two_waits = [] { asm volatile("s_nop 1"); };
    if constexpr (F8 && kMode != kLast) {
      op[0] = convert_k(ka[0]);
      converted(0);
      two_waits();
    }
    // ---- QK MFMAs of step st + 1; exponentials of the first 16 keys' pairs
    static_for<NQ>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
      if constexpr (kMode != kLast) {
        if constexpr (F8) diff_qk<DT, false, (c < 2)>(s_next[c % 2], op[c % 2], qv[c % 2][c / 2]);
        else qk(cc, s_next, ka[c]);
      }
      reads_at(cc);
      if constexpr (F8) {
        if constexpr (c + 1 == NQ) {
          op[0] = convert_v(0, va[0]);
          converted(0);
        } else if constexpr (kMode != kLast) {
          op[(c + 1) % 2] = convert_k(ka[c + 1]);
          converted((c + 1) % 2);
        }
        if constexpr (c * 8 / NQ == (c + 1) * 8 / NQ && (c == 0 || (c - 1) * 8 / NQ == c * 8 / NQ)) two_waits();
      }
#pragma unroll
      for (int q = c * 8 / NQ; q < (c + 1) * 8 / NQ; ++q) pair_exp(q);
      if constexpr (c > 0) {
#pragma unroll
        for (int q = (c - 1) * 8 / NQ; q < c * 8 / NQ; ++q) pair_pack(q);
      }
      sched_fence();
    });
    // ---- PV MFMAs of step st
    bool kfast = false, vfast = false;
    uint32_t kp0 = 0, kp1 = 0, vp0 = 0, vp1 = 0;
    if (kMode == kAny && jv < nsteps) {
      kp0 = __builtin_amdgcn_readfirstlane(pgk.x);
      kp1 = TPP == 16 ? __builtin_amdgcn_readfirstlane(pgk.y) : kp0;
      vp0 = __builtin_amdgcn_readfirstlane(pgv.x);
      vp1 = TPP == 16 ? __builtin_amdgcn_readfirstlane(pgv.y) : vp0;
      kfast = jk < nsteps && is_fast(jk, kp0, kp1);
      vfast = is_fast(jv, vp0, vp1);
    }
    Seen vis{0, 0};
    if constexpr (kMode == kAny) vis = seen(st + 1);
    float sc[2] = {0.f, 0.f}, bm[2] = {-INFINITY, -INFINITY};
    if constexpr (kMode != kLast) {
      sc[0] = score_scale(0, st + 1);
      sc[1] = F8 ? score_scale(1, st + 1) : sc[0];
    }
    constexpr int NPV = 2 * NQ;  // chunk c: operand c / 2, map c % 2
    static_for<NPV>([&](auto cc) {
      constexpr int c = decltype(cc)::value;
      constexpr int m = c / 2, r = c % 2, ks = m / KS, t = m % KS;
      if constexpr (c < 2 * NC && kMode != kLast) {
        if constexpr (kMode == kFast) {
          if constexpr (c < NC) copy_k(c, jk, pgk.x, pgk.y);
          else copy_v(c - NC, jv, pgv.x, pgv.y);
        } else if constexpr (c < NC) {
          if (kfast) copy_k(c, jk, kp0, kp1);
        } else {
          if (vfast) copy_v(c - NC, jv, vp0, vp1);
        }
      }
      if constexpr (F8) {
        diff_mma<DT, false, r * KS + t>(op[m % 2], pp[r][ks][t / (KS / 2)]);
      } else {
        diff_mma<DT, true, r * KS + t>(va[m], pp[r][ks][0]);
      }
      reads_at(std::integral_constant<int, NQ + c>{});
      if constexpr (F8 && r == 1 && m + 1 < NQ) {
        op[(m + 1) % 2] = convert_v(m + 1, va[m + 1]);
        converted((m + 1) % 2);
        if constexpr (kMode == kLast) two_waits();
      }
      if constexpr (c == 0) {
        static_for<8>([&](auto qq) {
          constexpr int q = decltype(qq)::value;
          if constexpr (q >= (NQ - 1) * 8 / NQ) pair_pack(q);
        });
        sched_fence();
        two_waits();  // the next MFMA may multiply that pair
      }
      // first half: exponentials of the other 16 keys
      if constexpr (c < NQ) {
        static_for<8>([&](auto qq) {
          constexpr int q = decltype(qq)::value;
          if constexpr (q >= c * 8 / NQ && q < (c + 1) * 8 / NQ) pair_exp(8 + q);
          if constexpr (c > 0 && q >= (c - 1) * 8 / NQ && q < c * 8 / NQ) pair_pack(8 + q);
        });
      }
      if constexpr (kMode != kLast) {
        if constexpr (c >= NQ) {  // second half: the next step's exponents and maxima
          constexpr int x0 = (c - NQ) * 32 / NQ, x1 = (c - NQ + 1) * 32 / NQ;
          static_for<32>([&](auto xx) {
            constexpr int y = decltype(xx)::value;
            if constexpr (y >= x0 && y < x1) {
              constexpr int rr = y / 16, x = y % 16;
              float v = fmaf(s_next[rr][x], sc[rr], mb[rr]);
              if constexpr (kMode == kAny) v = place(x) < vis.of(x) ? v : -INFINITY;
              e_cur[rr][x] = v;
              bm[rr] = fmaxf(bm[rr], v);
            }
          });
        }
      }
      sched_fence();
      if constexpr (c == NQ - 1) {
        static_for<8>([&](auto qq) {
          constexpr int q = decltype(qq)::value;
          if constexpr (q >= (NQ - 1) * 8 / NQ) pair_pack(8 + q);
        });
        sched_fence();
        if constexpr (kMode == kLast) two_waits();
      }
    });
    if constexpr (kMode == kLast) {
      acc_settle();
    } else {
      if (__ballot(fmaxf(bm[0], bm[1]) > kLazyRescale)) {
        acc_settle();
        float scale[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool moves = max_xor32(bm[r]) > kLazyRescale;
          const float m_new = moves ? -step_max(kMode == kAny, vis, s_next[r], sc[r]) : mb[r];
          scale[r] = __builtin_amdgcn_exp2f(m_new - mb[r]);
          mb[r] = m_new;
          exponents(r, kMode == kAny, vis, s_next[r], sc[r]);
          l_run[r] *= scale[r];
        }
        static_for<2 * KS * 16>([&](auto x) {
          constexpr int X = decltype(x)::value;
          diff_acc_put<X>(diff_acc_get<X>() * scale[X / (KS * 16)]);
        });
        acc_settle();
      }
      if constexpr (kMode == kAny) {
        if (const int chunk = pid_chunk_to_stage(st, TPP, n_pid)) stage_pids(chunk);
        if (jv < nsteps) {
          if (jk < nsteps && !kfast) slow_k(jk, kp0, kp1);
          if (!vfast) slow_v(jv, vp0, vp1);
        }
      }
    }
  };
  using Fast = std::integral_constant<int, kFast>;
  using Any = std::integral_constant<int, kAny>;
  using Last = std::integral_constant<int, kLast>;
  const int n_main = min(nsteps - 1, min_lim / kKeys - 1);
  int st = 0;
  int staged_at = -2;  // the iteration that staged page ids last (its flag is read two iterations later)
  while (st < nsteps - 1) {
    const int chunk_st = pid_next_staging(st, TPP);
    const int fast_end = min(min(n_main, paged_full - kDiffLeadK), chunk_st);
    if (st < fast_end && st >= staged_at + 2 && __builtin_amdgcn_readfirstlane(L.lim[kBad]) == 0) {
      for (; st < fast_end; ++st) step(Fast{}, st);
    } else {
      if (st == chunk_st) staged_at = st;
      step(Any{}, st);
      ++st;
    }
  }
  if (nsteps > 0) {
    step(Last{}, st);
  } else {
    static_for<2 * KS * 16>([](auto x) { diff_acc_put<decltype(x)::value>(0.f); });
    acc_settle();
  }

  // ---- difference, norm and output: lane holds O_m[M-row col][32n + 8(x/4) + 4 half + x%4].
  // x goes into the first map's registers while its squares are summed; the rows
  // leave through LDS (the step buffers; 16-byte chunk c of row i at chunk c ^ i)
  // as whole rows.
  DiffArgs* out_args = diff_args();
  const int out_lane = lane_now(), out_col = out_lane & 31, out_half = out_lane >> 5;
  const bool claims = w == 0 && out_lane == 0 &&
                      static_cast<unsigned>(out_args->hdr[2]) * out_args->num_kv_heads * out_args->tile_chunks > gridDim.x;
  uint32_t claimed = 0;
  if (claims) claimed = atomicAdd(out_args->claim + uniform(L.tile[5]), 1u);
  const float l1 = sum_xor32(l_run[0]), l2 = sum_xor32(l_run[1]);
  const float f1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;  // (no score above -inf: the map adds nothing)
  const float f2 = l2 > 0.f || l2 != l2 ? -L.lam[row_ok ? my_h : 0] / l2 : 0.f;
  float ss[4] = {0.f, 0.f, 0.f, 0.f};
  static_for<KS * 16>([&](auto xc) {
    constexpr int X = decltype(xc)::value;
    diff_acc_join<X>(f1, diff_acc_mul<KS * 16 + X>(f2), ss[X % 4]);
  });
  float scale = 1.f;
  if (out_args->norm_weight)
    scale = 1.f / sqrtf(sum_xor32((ss[0] + ss[1]) + (ss[2] + ss[3])) * (1.f / VD) + out_args->norm_eps);
  __syncthreads();  // every wavefront has read the last step
  if (claims) {
    DiffArgs* p = diff_args();
    const unsigned items = static_cast<unsigned>(p->hdr[2]) * p->num_kv_heads * p->tile_chunks;
    uint32_t q = L.tile[5];
    unsigned next = diff_item_of(q, claimed, gridDim.x);
#pragma unroll 1
    for (int k = 1; k < kDiffQueues && next >= items; ++k) {  // that queue is empty: the next one with an item
      q = (q + 1) % kDiffQueues;
      next = diff_item_of(q, atomicAdd(p->claim + q, 1u), gridDim.x);
    }
    L.next[0] = next;
    L.next[1] = q;
    if (next < items) {
      const uint32_t* entry = diff_entry(p, next);
      L.next[2] = entry[0];
      L.next[3] = entry[1];
    }
  }
  constexpr int kCh = VD / 8;  // 16-byte chunks of a row
  auto place_chunk = [](int row, int c) { return (kCh & (kCh - 1)) == 0 ? c ^ (row & (kCh - 1)) : (c + row) % kCh; };
  static_assert(sizeof(L.k) + sizeof(L.v) >= 128 * VD * 2, "the step buffers hold the tile's rows");
  uint16_t* region = L.k + w * 32 * VD;
  static_for<KS * 4>([&](auto qc) {
    constexpr int c = decltype(qc)::value;  // dims 8c + 4 half .. +3
    constexpr int x = 16 * (c / 4) + 4 * (c % 4);
    const f32x4 wt = *reinterpret_cast<const f32x4*>(L.weight + 8 * c + 4 * out_half);
    const float y0 = diff_acc_mul<x>(scale) * wt[0], y1 = diff_acc_mul<x + 1>(scale) * wt[1];
    const float y2 = diff_acc_mul<x + 2>(scale) * wt[2], y3 = diff_acc_mul<x + 3>(scale) * wt[3];
    *reinterpret_cast<u32x2*>(region + out_col * VD + place_chunk(out_col, c) * 8 + 4 * out_half) =
        u32x2{Dt<DT>::pack2(y0, y1), Dt<DT>::pack2(y2, y3)};
  });
  compiler_fence();
  __builtin_amdgcn_s_waitcnt(kLgkmZero);  // a wavefront reads only what it wrote
  compiler_fence();
  const int out_tile_heads = out_args->tile_heads, out_heads = out_args->num_q_heads / 2, out_qt = out_args->tile_rows;
  const int out_rows = uniform(L.tile[1]), out_hg = uniform(L.tile[4]);
  uint16_t* out_tile = out_args->out + (static_cast<int64_t>(uniform(L.tile[0])) * out_heads + uniform(L.tile[2]) * out_args->group +
                                        uniform(L.tile[3])) * VD;
#pragma unroll
  for (int it = 0; it < kCh / 2; ++it) {
    const int i = it * kWave + out_lane;
    const int row = i / kCh, c = i % kCh;
    const int m = w * 32 + row;
    const int t = static_cast<int>((static_cast<uint32_t>(m) * out_args->tile_magic) >> 16);
    const int h = m - t * out_tile_heads;
    const u32x4 val = *reinterpret_cast<const u32x4*>(region + row * VD + place_chunk(row, c) * 8);
    if (t < out_rows && t < out_qt && h < out_hg)
      *reinterpret_cast<u32x4*>(out_tile + (static_cast<int64_t>(t) * out_heads + h) * VD + c * 8) = val;
  }
}

template <int DT, int HD, int TPP, bool KV8>
__global__ __launch_bounds__(kPfThreads) PAL_DIFF_TILE_KERNEL void diff_tile_kernel(const DiffParams) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tile_lds[];
  DiffTileLds<HD, KV8>& L = *reinterpret_cast<DiffTileLds<HD, KV8>*>(tile_lds);
  unsigned item = blockIdx.x;
  uint32_t queue = item % kDiffQueues;
  {
    DiffArgs* p = diff_args();
    if (item >= static_cast<unsigned>(p->hdr[2]) * p->num_kv_heads * p->tile_chunks) return;
  }
  const uint32_t* entry = diff_entry(diff_args(), item);
  uint32_t row0 = __builtin_amdgcn_readfirstlane(entry[0]), seq = __builtin_amdgcn_readfirstlane(entry[1]);
  for (;;) {
    diff_tile<DT, HD, TPP, KV8>(item, queue, static_cast<int>(row0), seq, L);
    DiffArgs* p = diff_args();
    const unsigned items = static_cast<unsigned>(p->hdr[2]) * p->num_kv_heads * p->tile_chunks;
    if (items <= gridDim.x) return;
    __syncthreads();
    item = __builtin_amdgcn_readfirstlane(L.next[0]);
    if (item >= items) return;
    queue = __builtin_amdgcn_readfirstlane(L.next[1]);
    row0 = __builtin_amdgcn_readfirstlane(L.next[2]);
    seq = __builtin_amdgcn_readfirstlane(L.next[3]);
  }
}

}  // namespace
}  // namespace pal
