// Differential attention of single rows (decode rows) over the paged cache: the
// device code of the stream over the cache and of the merge behind it.
//
// For output head i with maps 1, 2 (query heads 2i, 2i + 1) and kv pair j (kv
// heads 2j, 2j + 1: two neighbouring (page, kv head) blocks of either pool):
//   O_m = sum_t e^(s_m,t - M_m) V_t,  l_m = sum_t e^(s_m,t - M_m),  s_m = q_m K_m^T / sqrt(HD)
//   x = O_1 / l_1 - lambda O_2 / l_2,  y = out_scale w x / sqrt(mean(x^2) + eps)
// in one pass over the keys with running maxima, the two maps' states apart
// (their exp-sums' ratio is known only at the end).
//
// Mapping: ordinary decode's (decode.hip), with the pair for the kv head.  The
// list of all 16-token blocks of the batch is cut into equal shares, one per
// resident wavefront; a wavefront streams its blocks with the loads of the next
// ones in flight, and split segments leave partials.  What differs:
//  * Up to 8 output heads of a kv pair are the 16 columns of the products:
//    columns 0..7 their first maps, 8..15 their second.  Both keys are multiplied
//    with all columns and each lane keeps the product that is its map's: as many
//    MFMAs as ordinary decode has for two kv heads, and an infinite key of one
//    map cannot reach the other (as zero-padded queries of 2 HD dims would let
//    it).  The value's 2 HD rows are then read once for both maps.
//  * The maps of a head sit in lanes r and r ^ 8, so the difference of a finished
//    segment is one lane rotation per value, and the norm's sum stays in the
//    wavefront.
//  * The probabilities enter the product with the values as two 16-bit terms, so
//    rounding them costs nothing of the result (see diff_range).
//  * Partials hold O, its maximum and exp-sum in fp32: the difference of two maps
//    may be small against either, and a partial rounded to 16 bits, as ordinary
//    decode keeps it, would cost 2^-8 of the maps.
//
// Measured (HD 128, 16-token pages unless said): 64 x 512-4,096 keys, 4 pairs of 4
// heads, stream 104 us (5.7 TB/s; HBM bounds it) and merge 8 us; fp8 pages 62 us
// (4.8 TB/s: the loads of one wavefront per SIMD bound it); 1,000 x 1-256 keys, 8
// pairs of 1 head, 197 us (5.3 TB/s); 4 x 32,768-131,072 keys of HD 64 in 32-token
// pages 97 us (5.6 TB/s) and merge 11 us.
#pragma once

#include "decode_plan.h"

namespace pal {
namespace {

constexpr int kDiffWaves = 4;  // independent wavefront workers per workgroup
constexpr int kDiffThreads = kDiffWaves * kWave;
constexpr int kDiffQueues = 8;       // claim counters of the tiles
// What a segment costs a worker beyond its blocks, in blocks: the last group of
// steps filled up, the segment's end.  Shares are cut from the blocks with so many
// empty ones behind each segment; cut from the blocks alone, a worker of short
// segments had twice the steps of the mean (1,000 x 1-256 keys, 16 kv heads:
// 261 us, now 197).
constexpr int kDiffSegmentCost = 3;
constexpr float kDiffLazyMax = 8.f;  // log2 headroom before a running max moves

// Up to kInlinePlanSeqs items of a batch, in LDS.
struct DiffPlanLds {
  int64_t cum[kInlinePlanSeqs + 1];
  int32_t len[kInlinePlanSeqs];
  int32_t seq[kInlinePlanSeqs];
  int32_t row[kInlinePlanSeqs];
  int64_t wave_sums[kDiffWaves];
};

// The plan of a mixed batch's rows, by one workgroup of T threads: the lone rows
// (alone in their run of rows of one sequence) with keys, and the tiles of the
// longer runs, each run cut from its first row on.  More tiles than the card
// takes at once are put in order of falling work (the keys of their first row),
// so that the last ones to start are short: 8 chunks of 512-2,048 rows on
// 0-2,048 cached, mean end of the workgroups 412 us, last 483 us without.  (A
// counting sort; equal tiles fall in any order, which changes no result.)  Lone
// rows without keys get their zeros.
//
// One compute unit runs all of it, so its time is the instructions per row: the
// rows are only searched for the starts of runs (ballots over groups of 64 rows,
// loads a sweep ahead), and what follows works on the runs found.  16 us for 10,344
// rows, 8 us for 2,052; with every row scanned for all three in code of 42 KB, whose
// first fetch takes most of it, 45 us and 41 us.
constexpr int kSortTiles = 4096;    // tiles put in order, at most (more: as they come)
constexpr int kTileBuckets = 1024;  // of a step of 32 keys, or more for page tables past 32,768 keys
constexpr int kPlanRows = 4;        // groups of a wavefront in a sweep
constexpr int kPlanRuns = 6144;     // starts of runs kept: a sweep's (4,096), and of some before it
template <int T>
struct DiffRowsLds {
  uint32_t start[kTileBuckets];
  u32x2 tile[kSortTiles];
  union {
    uint32_t run[kPlanRuns];
    uint16_t key[kSortTiles];
  };
  int64_t sums[T / kWave];
  int64_t total[2];
  uint32_t found[T / kWave];
};
template <int T, int kPer, int HD, int TPP>
__device__ __forceinline__ void diff_plan_rows(const DiffParams& p, DiffRowsLds<T>& L, bool keep_lone) {
  constexpr int kWaves = T / kWave;
  static_assert(T * kPer < kPlanRuns);
  const int tid = threadIdx.x;
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t n = static_cast<uint32_t>(p.num_seqs);
  const int64_t max_tokens = p.page_table_width * TPP;
  const int64_t segs = static_cast<int64_t>(p.num_kv_heads) * p.head_chunks;
  auto keys_of = [&](uint32_t sq, uint32_t r) {
    if (sq >= p.num_pt_rows) return static_cast<int64_t>(0);
    const int64_t off = p.q_offset[r], all = p.seq_lens[sq];
    const int64_t k = off < all ? off : all;
    PAL_DEBUG_FLAG(k > max_tokens, kDebugLength);
    return k < 0 ? static_cast<int64_t>(0) : (k > max_tokens ? max_tokens : k);
  };
  const uint64_t lower = (1ull << lane) - 1;  // the lanes before this one
  // rows of a wavefront: as few groups as hold the batch
  const uint32_t need = (n + T - 1) / T;
  const uint32_t groups = need < kPer ? need : kPer;
  uint32_t n_lone = 0, n_tiles = 0, n_runs = 0;  // so far; runs in L.run
  int64_t n_blocks = 0;
  uint32_t sq[kPer], edge;  // loaded a sweep ahead: the wavefront's rows, the row before them
  auto load = [&](uint32_t w0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t r = w0 + k * kWave + lane;
      sq[k] = static_cast<uint32_t>(k) < groups && r < n ? p.q2seq[r] : 0u;
    }
    edge = w0 > 0 && w0 <= n ? p.q2seq[w0 - 1] : 0u;
  };
  load(static_cast<uint32_t>(w) * kWave * groups);
#pragma unroll 1
  for (uint32_t base = 0; base < n; base += T * groups) {
    const uint32_t w0 = base + static_cast<uint32_t>(w) * kWave * groups;
    uint64_t starts[kPer];
    uint32_t prev = edge, mine = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t r = w0 + k * kWave + lane;
      uint32_t left = __shfl_up(sq[k], 1, kWave);
      if (lane == 0) left = prev;
      prev = __builtin_amdgcn_readlane(sq[k], kWave - 1);
      starts[k] = __ballot(static_cast<uint32_t>(k) < groups && r < n && (r == 0 || left != sq[k]));
      mine += __builtin_popcountll(starts[k]);
    }
    load(w0 + T * groups);
    if (lane == 0) L.found[w] = mine;
    __syncthreads();
    uint32_t at = n_runs;
    for (int i = 0; i < kWaves; ++i) {
      const uint32_t f = L.found[i];
      at += i < w ? f : 0u;
      n_runs += f;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      if (starts[k] >> lane & 1) L.run[at + __builtin_popcountll(starts[k] & lower)] = w0 + k * kWave + lane;
      at += __builtin_popcountll(starts[k]);
    }
    __syncthreads();
    const bool end = base + T * groups >= n;
    if (!end && n_runs + T * groups <= kPlanRuns) continue;
    // The runs with a known end: all at the end of the rows, else all but the last.
    const uint32_t done = end ? n_runs : n_runs - 1;
#pragma unroll 1
    for (uint32_t j = 0; j < done; j += T) {
      const uint32_t i = j + tid;
      const bool in = i < done;
      const uint32_t row = in ? L.run[i] : 0u;
      const uint32_t rows = in ? (i + 1 < n_runs ? L.run[i + 1] : n) - row : 0u;
      const uint32_t seq = in ? p.q2seq[row] : 0u;
      int64_t keys = 0;
      if (rows == 1 && keep_lone) {
        keys = keys_of(seq, row);
        if (keys == 0) zero_item_output<HD>(p, row);
      }
      const uint32_t tiles = rows > 1 ? (__umulhi(rows - 1, p.rows_magic) >> p.rows_shift) + 1 : 0u;
      const int64_t count = static_cast<int64_t>(keys > 0) << 32 | tiles;
      const int64_t count_to = block_inclusive_scan<T>(count, L.sums);
      const int64_t blocks = keys > 0 ? (((keys + 15) >> 4) + kDiffSegmentCost) * segs : 0;
      const int64_t blocks_to = keep_lone ? block_inclusive_scan<T>(blocks, L.sums) : 0;
      if (tid == T - 1) {
        L.total[0] = count_to;
        L.total[1] = blocks_to;
      }
      if (keys > 0) {
        const int64_t li = n_lone + static_cast<uint32_t>((count_to - count) >> 32);
        *reinterpret_cast<u32x4*>(p.lone + 4 * li) = u32x4{row, seq, static_cast<uint32_t>(keys), 0u};
        p.cum[li] = n_blocks + blocks_to - blocks;
      }
      auto put = [&](uint32_t i, uint32_t row, uint32_t seq) {
        const u32x2 t = {row, seq};
        if (i < kSortTiles)
          L.tile[i] = t;
        else
          *reinterpret_cast<u32x2*>(p.tiles + 2 * static_cast<int64_t>(i)) = t;
      };
      const uint32_t ti = n_tiles + static_cast<uint32_t>(count_to - count);
      if (tiles == 1) put(ti, row, seq);
      for (uint64_t more = __ballot(tiles > 1); more; more &= more - 1) {  // longer runs: by the wavefront
        const int l = __builtin_ctzll(more);
        const uint32_t c = __builtin_amdgcn_readlane(tiles, l), t0 = __builtin_amdgcn_readlane(ti, l);
        const uint32_t r0 = __builtin_amdgcn_readlane(row, l), sq0 = __builtin_amdgcn_readlane(seq, l);
        for (uint32_t m = lane; m < c; m += kWave) put(t0 + m, r0 + m * p.tile_rows, sq0);
      }
      __syncthreads();
      n_lone += static_cast<uint32_t>(L.total[0] >> 32);
      n_tiles += static_cast<uint32_t>(L.total[0]);
      n_blocks += L.total[1];
      __syncthreads();
    }
    if (!end) {
      const uint32_t open = L.run[done];
      __syncthreads();
      if (tid == 0) L.run[0] = open;
      n_runs = 1;
    }
  }
  const int64_t items = static_cast<int64_t>(n_tiles) * p.num_kv_heads * p.tile_chunks;
  const bool sort = items > p.num_workers / kDiffWaves && n_tiles <= kSortTiles;
  if (tid == 0) {
    if (keep_lone) {
      p.hdr[0] = n_blocks;
      p.hdr[1] = n_lone;
      p.cum[n_lone] = n_blocks;
    }
    p.hdr[2] = n_tiles;
    p.hdr[3] = sort;
  }
  if (sort)
    for (int b = tid; b < kTileBuckets; b += T) L.start[b] = 0;
  __syncthreads();
  if (!sort) {  // in the rows' order
    for (uint32_t i = tid; i < n_tiles && i < kSortTiles; i += T)
      *reinterpret_cast<u32x2*>(p.tiles + 2 * i) = L.tile[i];
    return;
  }
  const int per_bucket = max(32, static_cast<int>((max_tokens + kTileBuckets - 1) / kTileBuckets));
  for (uint32_t i = tid; i < n_tiles; i += T) {
    const u32x2 t = L.tile[i];
    const uint32_t b = static_cast<uint32_t>(keys_of(t.y, t.x)) / static_cast<uint32_t>(per_bucket);
    const uint32_t key = kTileBuckets - 1 - (b < kTileBuckets - 1 ? b : kTileBuckets - 1);
    L.key[i] = static_cast<uint16_t>(key);
    atomicAdd(&L.start[key], 1u);
  }
  __syncthreads();
  constexpr int kB = kTileBuckets / T;
  int64_t sum = 0;
#pragma unroll
  for (int k = 0; k < kB; ++k) sum += L.start[tid * kB + k];
  int64_t at = block_inclusive_scan<T>(sum, L.sums) - sum;
#pragma unroll
  for (int k = 0; k < kB; ++k) {
    const uint32_t c = L.start[tid * kB + k];
    L.start[tid * kB + k] = static_cast<uint32_t>(at);
    at += c;
  }
  __syncthreads();
  for (uint32_t i = tid; i < n_tiles; i += T)
    *reinterpret_cast<u32x2*>(p.tiles + 2 * atomicAdd(&L.start[L.key[i]], 1u)) = L.tile[i];
}

// The plan of more rows than a stream workgroup scans.
template <int HD, int TPP>
__global__ __launch_bounds__(kPlanThreads) void diff_plan_kernel(const DiffParams p) {
  __shared__ DiffRowsLds<kPlanThreads> L;
  diff_plan_rows<kPlanThreads, kPlanRows, HD, TPP>(p, L, true);
}

// x's value in lane l ^ 8 (a rotation by 8 of each 16 lanes)
__device__ __forceinline__ float lane_xor8(float x) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128, 0xf, 0xf, true));  // row_ror:8
}

// Streams the blocks of virtual worker v.  The blocks form a run of pieces (the
// blocks of one segment inside the worker's range); the pipeline runs through
// piece boundaries: while the last blocks of a piece are computed, the first
// of the next piece are loading (its item, query and first page ids were fetched
// when the piece before it started).
// Descriptor of `bytes` bytes at a wavefront's common address: loads past them
// read nothing and give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_descriptor(const uint8_t* at, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(at);
  // (the builtin returns an int: without the casts a low half past 2^31 would be sign-extended)
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32)));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0, bytes,
                                           0x00027000);
}

template <int DT, int HD, int TPP, int PF, bool KV8>
__device__ __forceinline__ void diff_range(const DiffParams& p, const Sched& sc, const int64_t* cum,
                                           const DiffPlanLds* plan, int64_t n_items, const float* weight, int64_t v) {
  static_assert(HD % 32 == 0 && (!KV8 || HD % 64 == 0), "whole k-steps and stripes");
  constexpr int KK = HD / 32;     // QK k-steps of 32 dims of one map
  constexpr int NT = 2 * HD / 16;  // output tiles of 16 dims
  constexpr int NBUF = PF + 1;
  constexpr int EB = KV8 ? 1 : 2;  // pool element bytes
  constexpr int KL = KV8 ? HD / 64 : KK;  // 16-byte key loads of one map
  // Type of the product with the values: fp8 codes are exact in bf16, whose range
  // holds a probability times any value scale (fp16's would lose small ones).
  using PV = Dt<KV8 ? kBF16 : DT>;

  const int64_t b0 = vstart(sc, v);
  const int64_t b_end = vstart(sc, v + 1);
  const int lane = lane_id();
  // the split segment whose first piece ends the worker's range, or none
  int64_t list_g0 = -1, list_nb = 0, list_row = 0, list_seg = 0;
  auto write_list = [&] {
    if (lane == 0) {
      int64_t* slot = p.split_list + 4 * v;
      slot[0] = list_g0;
      slot[1] = list_nb;
      slot[2] = list_row;
      slot[3] = list_seg;
    }
  };
  if (b_end <= b0) {
    write_list();
    return;
  }

  const int g = lane >> 4;
  const int r16 = lane & 15;
  const int map = r16 >> 3;  // this lane's column: map, and head of the chunk
  const int r8 = r16 & 7;
  const int segs = p.num_kv_heads * p.head_chunks;
  const int64_t head_block = static_cast<int64_t>(HD) * TPP * EB;  // bytes per (page, kv head)
  const int64_t page_stride = head_block * 2 * p.num_kv_heads;

  // A piece: item s (row `row` of page-table row `seq`, `len` keys, nb blocks per segment),
  // segment `seg`, blocks [blk, blk + count) of the segment, from global block
  // gpos on; r = its place in the units of the item (a segment has nb +
  // kDiffSegmentCost of them, as the global list has).  c_* is
  // the piece being computed, x_* the next one (kept in scalars).
  int64_t c_s, c_r, c_gpos, c_row, c_seq, c_len, c_nb, c_blk, c_count;
  int c_seg;
  int64_t x_s, x_r, x_gpos, x_row, x_seq, x_len, x_nb, x_blk, x_count;
  int x_seg;
#define PAL_FIND_PIECE(P, S0, R0, G0)                                                      \
  do {                                                                                     \
    int64_t s_ = (S0), r_ = (R0), g_ = (G0), len_, seq_, row_, nb_, unit_, seg_ = 0, blk_ = 0; \
    for (;;) {                                                                             \
      if (plan) {                                                                          \
        len_ = plan->len[s_];                                                              \
        seq_ = plan->seq[s_];                                                              \
        row_ = plan->row[s_];                                                              \
      } else if (p.q2seq) {                                                                \
        row_ = p.lone[4 * s_];                                                             \
        seq_ = p.lone[4 * s_ + 1];                                                         \
        len_ = p.lone[4 * s_ + 2];                                                         \
      } else {                                                                             \
        const Item it_ = item_at(p, s_, TPP);                                              \
        len_ = it_.len;                                                                    \
        seq_ = it_.seq;                                                                    \
        row_ = s_;                                                                         \
      }                                                                                    \
      nb_ = (len_ + 15) >> 4;                                                              \
      unit_ = nb_ + kDiffSegmentCost;                                                      \
      if (len_ > 0) {                                                                      \
        seg_ = r_ / unit_;                                                                 \
        blk_ = r_ - seg_ * unit_;                                                          \
        if (blk_ < nb_) break;                                                             \
        r_ += unit_ - blk_; /* behind a segment: on to the next */                         \
        g_ += unit_ - blk_;                                                                \
        if (g_ >= b_end) break;                                                            \
        if (r_ < unit_ * segs) continue;                                                   \
      }                                                                                    \
      ++s_;                                                                                \
      r_ = 0;                                                                              \
    }                                                                                      \
    P##s = s_;                                                                             \
    P##r = r_;                                                                             \
    P##gpos = g_;                                                                          \
    P##row = row_;                                                                         \
    P##seq = seq_;                                                                         \
    P##len = len_;                                                                         \
    P##nb = nb_;                                                                           \
    P##seg = static_cast<int>(seg_);                                                       \
    P##blk = blk_;                                                                         \
    P##count = (P##nb - P##blk) < (b_end - P##gpos) ? (P##nb - P##blk) : (b_end - P##gpos); \
  } while (0)

  // Q^T operand of a piece: the dims of this lane's k-slices of its column's
  // query (zeros in columns without a head).
  // Its lambda comes with it: a load at the piece's end would wait for the next
  // piece's blocks, in flight by then.
  u32x4 qv[KK], qn[KK];
  float lam, lam_n;
  auto load_q = [&](int64_t row, int seg, u32x4 (&q)[KK], float& l) {
    const int h0 = (seg % p.head_chunks) * 8;
    const bool hv = r8 < min(8, p.group - h0);
    const uint32_t qmask = hv ? 0xFFFFFFFFu : 0u;
    const int64_t head = static_cast<int64_t>(seg / p.head_chunks) * p.group + h0 + (hv ? r8 : 0);
    const uint16_t* qrow = p.q + (row * p.num_q_heads + 2 * head + map) * HD;
    l = p.lambdas[head];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      if constexpr (KV8)  // k-step kk = (stripe g + 4 (kk / 2), half kk % 2)
        q[kk] = *reinterpret_cast<const u32x4*>(qrow + 16 * (g + 4 * (kk >> 1)) + 8 * (kk & 1)) & qmask;
      else
        q[kk] = *reinterpret_cast<const u32x4*>(qrow + 32 * kk + 8 * g) & qmask;
    }
  };
  // page ids of window wi (64 pages, one per lane) of a piece
  auto load_window = [&](int64_t seq, int64_t blk, int64_t wi) {
    const uint32_t* pt = p.page_table + seq * p.page_table_width;
    int64_t lp = (blk * 16) / TPP + wi * kWave + lane;
    if (lp >= p.page_table_width) lp = p.page_table_width - 1;
    return pt[lp];
  };
  {
    const int64_t s0 = locate_seq(cum, n_items, b0);  // the item holding block b0 (it has blocks)
    PAL_FIND_PIECE(c_, s0, b0 - cum[s0], b0);
  }
  if (c_gpos >= b_end) {  // the range lies behind a segment
    write_list();
    return;
  }
  load_q(c_row, c_seg, qv, lam);

  // Page ids in register windows of 64 pages: pid_cur holds window wcur, the
  // window of the block being computed, pid_nxt the next one; every step group
  // also loads the one after that, and the windows move up when the computed
  // block enters window wcur + 1.
  int wcur = 0;
  uint32_t pid_cur = load_window(c_seq, c_blk, 0), pid_nxt = load_window(c_seq, c_blk, 1),
           pid_later = load_window(c_seq, c_blk, 2);

  u32x4 kb[NBUF][2][KL];
  u32x2 vb[NBUF][KV8 ? 1 : NT];
  u32x4 vq8[NBUF][KV8 ? NT / 4 : 1];
  f32x2 bks[NBUF], bvs[NBUF];  // fp8: the block's scales, of kv heads 2j and 2j + 1
  bool bv[NBUF];

  bool prologue = true;  // the pipeline is empty
  bool has_next = false;
  x_s = c_s; x_r = c_r; x_gpos = c_gpos; x_row = c_row; x_seq = c_seq; x_len = c_len; x_nb = c_nb; x_blk = c_blk;
  x_count = c_count; x_seg = c_seg;
  uint32_t pidn0 = 0;        // window 0 of the next piece (a load in flight)
  uint32_t pidn0_ready = 0;  // the same once it has arrived (see below)

  for (;;) {
    const int pair = c_seg / p.head_chunks;
    const int h0 = (c_seg % p.head_chunks) * 8;
    const int hg = min(8, p.group - h0);
    const bool complete = (c_blk == 0) && (c_count == c_nb);
    const int len = static_cast<int>(c_len);
    const int n_blk = static_cast<int>(c_count);
    const int n_pad = (n_blk + NBUF - 1) / NBUF * NBUF;  // steps of the piece
    const int bstart = static_cast<int>(c_blk);
    const int pbase = (bstart * 16) / TPP;
    const uint8_t* kbase = static_cast<const uint8_t*>(p.k_pool) + pair * 2 * head_block;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v_pool) + pair * 2 * head_block;
    const uint8_t* kbase_n = kbase;  // set once the next piece is known
    const uint8_t* vbase_n = vbase;
    int pair_n = pair;
    int nblk_n = 1;
    int bstart_n = 0, pbase_n = 0;

    // Issues the loads of step i of the piece into buffer `buf`: block i of the
    // piece or, past the piece's steps, block i - n_pad of the next piece.  They go
    // through descriptors of the pair's block: a step past the piece's end, or with
    // a page id out of range, takes one of no bytes, whose loads read no memory and
    // give zeros (the block is masked when computed).  Every block is read once per
    // call: non-temporal, but for 32-token pages, whose rows this block and the
    // next share (as in ordinary decode: cacheable where a kv head's block holds
    // 8 KiB or more).
    constexpr int kPolicy = TPP == 32 && 2 * HD * TPP * EB >= 8192 ? 0 : 2;  // 2: non-temporal
    auto issue = [&](int i, int buf, uint32_t w_n0) {
      const bool to_next = has_next && i >= n_pad;
      const int j = to_next ? i - n_pad : i;
      const int b = (to_next ? bstart_n : bstart) + j;
      const int e = (b * 16) / TPP - (to_next ? pbase_n : pbase);  // page within the piece's windows
      // (selects of values: a select of two variables' addresses would push the
      // pipeline state to scratch)
      const uint32_t w_c = pid_cur, w_x = pid_nxt;
      const uint32_t win = to_next ? w_n0 : ((e >> 6) == wcur ? w_c : w_x);
      const uint32_t pg = __builtin_amdgcn_readlane(win, static_cast<int>(e & 63));
      bv[buf] = pg < p.num_pages;
      const bool in = j < (to_next ? nblk_n : n_blk);
      PAL_DEBUG_FLAG(!bv[buf] && in, kDebugPageId);
      const bool ok = __builtin_amdgcn_readfirstlane(bv[buf] && in);
      const uint32_t page = ok ? pg : 0u;
      const uint32_t slot0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>((b * 16) % TPP));
      const uint8_t* kb_x = kbase_n;
      const uint8_t* vb_x = vbase_n;
      const int bytes = ok ? static_cast<int>(2 * head_block) : 0;
      const auto kd = block_descriptor((to_next ? kb_x : kbase) + static_cast<int64_t>(page) * page_stride, bytes);
      const auto vd = block_descriptor((to_next ? vb_x : vbase) + static_cast<int64_t>(page) * page_stride, bytes);
      if constexpr (KV8) {
        const int64_t si = 2 * (static_cast<int64_t>(page) * p.num_kv_heads + (to_next ? pair_n : pair));
        bks[buf] = f32x2{p.k_scales[si], p.k_scales[si + 1]};
        bvs[buf] = f32x2{p.v_scales[si], p.v_scales[si + 1]};
      }
      // (the empty asm keeps the sums with constants here, where they become the loads' offsets)
      uint32_t k_at = (r16 + g * TPP) * 16;
      uint32_t v_at = KV8 ? (16 * g + r16) * TPP : (r16 * TPP + 4 * g) * 2;
      asm volatile("" : "+v"(k_at), "+v"(v_at));
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int kk = 0; kk < KL; ++kk)
          kb[buf][a][kk] = __builtin_amdgcn_raw_buffer_load_b128(
              kd, k_at + a * (HD * TPP * EB) + 4 * kk * TPP * 16, slot0 * 16, kPolicy);
      if constexpr (KV8) {
        // lane 16g + i reads the block's 16 codes of dim row 64q + 16g + i; compute
        // transposes them across the lane groups
#pragma unroll
        for (int q = 0; q < NT / 4; ++q)
          vq8[buf][q] = __builtin_amdgcn_raw_buffer_load_b128(vd, v_at + 64 * q * TPP, slot0, kPolicy);
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          vb[buf][n] = __builtin_amdgcn_raw_buffer_load_b64(vd, v_at + 32 * n * TPP, slot0 * 2, kPolicy);
      }
    };

    float m_run = -INFINITY;  // running max of this lane's column (log2 units)
    float l_run = 0.f;        // this lane's share of its exp-sum
    f32x4 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto compute = [&](int i, int buf) {
      const int b = bstart + i;
      const bool live = bv[buf] && i < n_blk;  // steps past the piece end are fully masked
      f32x4 acc[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        acc[a] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          if constexpr (KV8) {
            const u32x4 w = kb[buf][a][kk / 2];
            acc[a] = Dt<DT>::mma16x16x32(fp8x8_exact<DT>(kk % 2 ? u32x2{w.z, w.w} : u32x2{w.x, w.y}), qv[kk], acc[a]);
          } else {
            acc[a] = Dt<DT>::mma16x16x32(kb[buf][a][kk], qv[kk], acc[a]);
          }
        }
      }
      const float ks = KV8 ? (map ? bks[buf].y : bks[buf].x) * p.scale_log2 : p.scale_log2;
      // tokens past the end (and whole invalid blocks) are masked: token 4g + e of
      // the block is a key when e < kl
      const int left = live ? len - b * 16 : 0;
      const int kl = static_cast<int>(left < 16 ? left : 16) - 4 * g;
      float sc4[4];
      float bm = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float s = (map ? acc[1][e] : acc[0][e]) * ks;
        sc4[e] = e < kl ? s : -INFINITY;
        bm = fmaxf(bm, sc4[e]);
      }
      // the running max of a column moves only when a score passes it by more
      // than the headroom (always for its first score above -inf)
      if (__ballot(bm > m_run + kDiffLazyMax)) {
        const float m_new = fmaxf(m_run, max_xor32(max_xor16(bm)));
        const float alpha = (m_new == -INFINITY) ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n] *= alpha;
        m_run = m_new;
      }
      const float mref = (m_run == -INFINITY) ? 0.f : m_run;
      float pe[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pe[e] = __builtin_amdgcn_exp2f(sc4[e] - mref);
        l_run += pe[e];
      }
      // The probabilities (fp8: times the value scale of the half's kv head; the
      // exp-sum takes them unscaled) go into the product as two 16-bit terms,
      // the rounded value and what the rounding left.  A lane's k-slots of the
      // 32-deep MFMA are its 4 tokens twice, against the first and the second
      // terms; the 16-deep one, with rounded probabilities alone, takes as long.
      // bf16, 64 x 512-4,096 keys, error of the result 2.6e-3 -> 1.7e-3.
      u32x4 pb[KV8 ? 2 : 1];
#pragma unroll
      for (int hf = 0; hf < (KV8 ? 2 : 1); ++hf) {
        float t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = KV8 ? pe[e] * bvs[buf][hf] : pe[e];
        const uint32_t w0 = PV::pack2(t[0], t[1]), w1 = PV::pack2(t[2], t[3]);
        pb[hf] = u32x4{w0, w1, PV::pack2(t[0] - PV::lo(w0), t[1] - PV::hi(w0)),
                       PV::pack2(t[2] - PV::lo(w1), t[3] - PV::hi(w1))};
      }
      // slots past the end may hold anything, NaN bits included: zero their values
      const uint32_t mlo = (kl > 0 ? 0x0000FFFFu : 0u) | (kl > 1 ? 0xFFFF0000u : 0u);
      const uint32_t mhi = (kl > 2 ? 0x0000FFFFu : 0u) | (kl > 3 ? 0xFFFF0000u : 0u);
      const uint32_t m8 = kl >= 4 ? 0xFFFFFFFFu : (kl <= 0 ? 0u : (0xFFFFFFFFu >> (32 - 8 * kl)));
      u32x4 vt[KV8 ? NT / 4 : 1];
      if constexpr (KV8) {
#pragma unroll
        for (int q = 0; q < NT / 4; ++q) vt[q] = transpose_lane_groups4(vq8[buf][q]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        u32x2 vv;
        if constexpr (KV8) {
          const uint32_t codes = vt[n >> 2][n & 3] & m8;  // a zero code is +0
          vv = u32x2{PV::fp8x2(codes, false), PV::fp8x2(codes, true)};
        } else {
          vv = u32x2{vb[buf][n].x & mlo, vb[buf][n].y & mhi};
        }
        o[n] = PV::mma16x16x32(u32x4{vv.x, vv.y, vv.x, vv.y}, pb[KV8 ? n / (NT / 2) : 0], o[n]);
      }
    };

    // The first piece fills the pipeline; a later one finds its first PF blocks
    // in flight.
    if (prologue) {
#pragma unroll
      for (int q = 0; q < PF; ++q) issue(q, q, pidn0);  // (never the next piece)
    }

    // The next piece: its item, query and first page ids load now, while this
    // piece streams (with none, the current one's again: no load under a branch).
    {
      const int64_t past = c_count + (c_blk + c_count == c_nb ? kDiffSegmentCost : 0);
      const int64_t gpos_n = c_gpos + past;
      has_next = gpos_n < b_end;
      int64_t s_n = c_s, r_n = c_r + past;
      if (r_n >= (c_nb + kDiffSegmentCost) * segs) {
        ++s_n;
        r_n = 0;
      }
      if (has_next) {
        PAL_FIND_PIECE(x_, s_n, r_n, gpos_n);
      } else {
        x_s = c_s; x_r = c_r; x_gpos = c_gpos; x_row = c_row; x_seq = c_seq; x_len = c_len; x_nb = c_nb; x_blk = c_blk;
        x_count = c_count; x_seg = c_seg;
      }
      load_q(x_row, x_seg, qn, lam_n);
      pidn0 = load_window(x_seq, x_blk, 0);
    }
    const uint32_t pidn1 = load_window(x_seq, x_blk, 1);
    {
      pair_n = x_seg / p.head_chunks;
      kbase_n = static_cast<const uint8_t*>(p.k_pool) + pair_n * 2 * head_block;
      vbase_n = static_cast<const uint8_t*>(p.v_pool) + pair_n * 2 * head_block;
      nblk_n = static_cast<int>(x_count);
      bstart_n = static_cast<int>(x_blk);
      pbase_n = (bstart_n * 16) / TPP;
    }

    // Every step issues and computes unconditionally (steps past the end re-read
    // the last block and compute it fully masked), so the compiler's wait counts
    // stay exact and the blocks in flight are never drained early.  The groups of
    // a piece with two or more of them select the next piece's window from
    // pidn0_ready, refreshed at the end of each group where the wait is exact:
    // selecting pidn0 would wait for that load at the top of every group.
    auto step_group = [&](int i0, uint32_t w_n0) {
      const uint32_t pid_ahead = load_window(c_seq, c_blk, wcur + 2);
#pragma unroll
      for (int u = 0; u < NBUF; ++u) {
        const int i = i0 + u;
        issue(i + PF, (u + PF) % NBUF, w_n0);
        compute(i, u);
      }
      const int e_last = ((bstart + i0 + NBUF - 1) * 16) / TPP - pbase;
      const bool up = (e_last >> 6) > wcur;
      pid_cur = up ? pid_nxt : pid_cur;
      pid_nxt = up ? pid_later : pid_nxt;
      wcur += up ? 1 : 0;
      pid_later = pid_ahead;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) asm volatile("" ::"v"(qn[kk]));
      asm volatile("" ::"v"(pidn1));
      asm volatile("" ::"v"(lam_n));
      asm volatile("v_mov_b32 %0, %1" : "=v"(pidn0_ready) : "v"(pidn0));
    };
    if (n_pad == NBUF) {
      step_group(0, pidn0);
    } else {
      int i0 = 0;
      do {
        step_group(i0, pidn0_ready);
        i0 += NBUF;
      } while (i0 < n_pad);
    }

    // ---- finish the piece: exp-sum of the column over the 4 lane groups
    const float l = sum_xor32(sum_xor16(l_run));
    if (complete) {
      // x = O_1 / l_1 - lambda O_2 / l_2: each lane adds its map's term to that of
      // lane ^ 8, so both hold x; the norm sums it over the 4 lane groups
      const int64_t head = static_cast<int64_t>(pair) * p.group + h0 + (r8 < hg ? r8 : 0);
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // (no score above -inf: the map adds nothing)
      const float f = map ? -lam * inv : inv;
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float t = o[n][e] * f;
          o[n][e] = t + lane_xor8(t);
          ss += o[n][e] * o[n][e];
        }
      }
      float scale = 1.f;
      if (p.norm_weight) scale = 1.f / sqrtf(sum_xor32(sum_xor16(ss)) * (1.f / (2 * HD)) + p.norm_eps);
      if (r8 < hg) {
        // the two lanes of a head write half of its row each
        uint16_t* row = p.out + (c_row * (p.num_q_heads / 2) + head) * (2 * HD) + 4 * g;
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
          const int t = n + map * (NT / 2);
          f32x4 y = map ? o[n + NT / 2] : o[n];
          y *= scale * *reinterpret_cast<const f32x4*>(weight + 16 * t + 4 * g);
          *reinterpret_cast<u32x2*>(row + 16 * t) = u32x2{Dt<DT>::pack2(y[0], y[1]), Dt<DT>::pack2(y[2], y[3])};
        }
      }
    } else {
      if (r8 < hg) {
        const int64_t slot = ((v * 2 + (c_gpos == b0 ? 0 : 1)) * 2 + map) * p.hg_max + r8;
        float* po = p.part_o32 + slot * (2 * HD) + 4 * g;
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(po + 16 * n) = o[n];
        if (g == 0) *reinterpret_cast<f32x2*>(p.part_ml + slot * 2) = f32x2{m_run, l};
      }
      if (c_blk == 0) {  // the first piece of a split segment ends the worker's range
        list_g0 = c_gpos;
        list_nb = c_nb;
        list_row = c_row;
        list_seg = c_seg;
      }
    }
    prologue = false;
    if (!has_next) break;
    // the next piece becomes current: its first PF blocks are in flight, in
    // buffers 0 .. PF-1 (n_pad is a multiple of NBUF)
    c_s = x_s; c_r = x_r; c_gpos = x_gpos; c_row = x_row; c_seq = x_seq; c_len = x_len; c_nb = x_nb; c_blk = x_blk;
    c_count = x_count; c_seg = x_seg;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qv[kk] = qn[kk];
    lam = lam_n;
    wcur = 0;
    pid_cur = pidn0;
    pid_nxt = pidn1;
    pid_later = load_window(c_seq, c_blk, 2);
  }
  write_list();
#undef PAL_FIND_PIECE
}

template <int DT, int HD, int TPP, bool KV8>
__global__ __launch_bounds__(kDiffThreads) __attribute__((amdgpu_waves_per_eu(1, 1)))
void diff_stream_kernel(const DiffParams p) {
  __shared__ union {
    DiffPlanLds plan;
    DiffRowsLds<kDiffThreads> rows;
  } lds_all;
  // what a row is scaled with behind its norm (in LDS: see load_q)
  __shared__ __attribute__((aligned(16))) float weight[2 * HD];
  DiffPlanLds& lds = lds_all.plan;
  const int64_t n = p.num_seqs;
  const int tid = threadIdx.x;
  const bool scan = n <= kInlinePlanSeqs;
  constexpr int kPer = kInlinePlanSeqs / kDiffThreads;
  if (p.q2seq && scan && blockIdx.x + 1 == gridDim.x) {  // the workgroup behind the workers'
    diff_plan_rows<kDiffThreads, kPer, HD, TPP>(p, lds_all.rows, false);
    return;
  }
  if (blockIdx.x == 0 && tid < kDiffQueues) p.claim[tid] = 0;  // for the tiles, the launch behind
  if (tid < 2 * HD) weight[tid] = p.out_scale * (p.norm_weight ? p.norm_weight[tid] : 1.f);
  int64_t n_items = n, total;
  const int64_t* cum = p.cum;
  const DiffPlanLds* plan = nullptr;
  if (scan) {
    // every workgroup scans the lengths into LDS: thread t owns items 4t .. 4t+3,
    // whose loads are in flight together
    const int64_t segs = static_cast<int64_t>(p.num_kv_heads) * p.head_chunks;
    const int64_t max_tokens = p.page_table_width * TPP;
    const int first = tid * kPer;
    const int last = static_cast<int>(n) - 1;
    uint32_t seq[kPer];
    int64_t keys[kPer];
    bool skip[kPer] = {};
    if (p.q2seq) {
      uint32_t sq[kPer + 2];
      int32_t off[kPer];
#pragma unroll
      for (int k = 0; k < kPer + 2; ++k) sq[k] = p.q2seq[max(0, min(first + k - 1, last))];
#pragma unroll
      for (int k = 0; k < kPer; ++k) off[k] = p.q_offset[min(first + k, last)];
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int s = first + k;
        skip[k] = (s > 0 && sq[k] == sq[k + 1]) || (s < last && sq[k + 2] == sq[k + 1]);  // a tile's row
        const bool has = sq[k + 1] < p.num_pt_rows && !skip[k];
        seq[k] = has ? sq[k + 1] : 0u;
        const int32_t all = p.num_pt_rows ? p.seq_lens[seq[k]] : 0;
        keys[k] = has ? min(all, off[k]) : 0;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        seq[k] = static_cast<uint32_t>(first + k);
        keys[k] = p.seq_lens[min(first + k, last)];
      }
    }
    int64_t vals[kPer];
    int64_t tsum = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int s = first + k;
      const bool in = s <= last;
      PAL_DEBUG_FLAG(in && keys[k] > max_tokens, kDebugLength);
      const int64_t len = !in || keys[k] < 0 ? 0 : (keys[k] > max_tokens ? max_tokens : keys[k]);
      vals[k] = len > 0 ? (((len + 15) >> 4) + kDiffSegmentCost) * segs : 0;
      if (in) {
        lds.len[s] = static_cast<int32_t>(len);
        lds.seq[s] = static_cast<int32_t>(seq[k]);
        lds.row[s] = s;
        if (len == 0 && !skip[k] && blockIdx.x == 0) zero_item_output<HD>(p, s);
      }
      tsum += vals[k];
    }
    const int64_t incl = block_inclusive_scan<kDiffThreads>(tsum, lds.wave_sums);
    int64_t c = incl - tsum;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t s = static_cast<int64_t>(tid) * kPer + k;
      if (s < n) lds.cum[s] = c;
      c += vals[k];
    }
    if (tid == kDiffThreads - 1) lds.cum[n] = incl;
    __syncthreads();
    total = lds.cum[n];
    if (blockIdx.x == 0 && tid == 0) p.hdr[0] = total;
    plan = &lds;
  } else {
    total = p.hdr[0];
    if (p.q2seq) {  // the lone rows that the plan found
      n_items = p.hdr[1];
      if (total > 0 && n_items <= kInlinePlanSeqs) {
        for (int64_t s = tid; s < n_items; s += kDiffThreads) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(p.lone + 4 * s);
          lds.row[s] = static_cast<int32_t>(v.x);
          lds.seq[s] = static_cast<int32_t>(v.y);
          lds.len[s] = static_cast<int32_t>(v.z);
          lds.cum[s] = p.cum[s];
        }
        __syncthreads();
        plan = &lds;
      }
    }
  }
  if (plan) cum = plan->cum;
  __syncthreads();
  if (total == 0) return;
  const Sched sc = make_sched(total, p.num_workers, 0);
  const int64_t w = static_cast<int64_t>(blockIdx.x) * kDiffWaves + wave_id();
  if (w < sc.nws) diff_range<DT, HD, TPP, KV8 ? 3 : 2, KV8>(p, sc, cum, plan, n_items, weight, w);
}

// Joins the pieces of split segments: workgroup (v, h) takes head h of the
// segment in list slot v, whose first piece is worker v's, further pieces the
// first ones of workers v + 1, v + 2, ...  A wavefront takes every fourth piece
// (times the rows one 16-byte load per lane covers), all maxima first (the first
// rows load beside them, as the lambda and the weight do: the kernel's time is
// its chain of loads):
//   O_m = sum_c 2^(M_c - M) O_c,  l_m = sum_c 2^(M_c - M) l_c
// the wavefronts' sums meet in LDS, and the first finishes the row.
template <int DT, int HD>
__global__ __launch_bounds__(kDiffThreads) void diff_merge_kernel(const DiffParams p) {
  constexpr int D = 2 * HD;
  constexpr int kLpr = D <= 64 ? 16 : (D <= 128 ? 32 : 64);  // lanes per partial row, 4 dims each
  constexpr int kRows = kWave / kLpr;                        // rows of one load
  constexpr int kBatch = 4;
  __shared__ __attribute__((aligned(16))) float sum_lds[kDiffWaves][2][D];
  __shared__ float l_lds[kDiffWaves][2];
  const int64_t e = blockIdx.x;
  const int h = blockIdx.y;
  const int64_t total = p.hdr[0];
  const int64_t* slot = p.split_list + 4 * e;
  const int64_t g0 = slot[0], nb = slot[1], row = slot[2];
  const int seg = static_cast<int>(slot[3]);
  if (total == 0) return;
  const Sched sc = make_sched(total, p.num_workers, 0);
  if (e >= sc.nws || g0 < 0) return;
  const int h0 = (seg % p.head_chunks) * 8;
  if (h >= min(8, p.group - h0)) return;
  const int head = (seg / p.head_chunks) * p.group + h0 + h;
  const int nc = static_cast<int>(vworker_of(sc, g0 + nb - 1) - e) + 1;
  const int t0 = vstart(sc, e) == g0 ? 0 : 1;  // the first piece's partial slot: 0 where the range starts with it
  const int lane = lane_id();
  const int w = wave_id();
  const int rl = lane % kLpr;
  const int rg = lane / kLpr;
  const bool dl = 4 * rl < D;
  auto row_of = [&](int c, int map) { return (((e + c) * 2 + (c == 0 ? t0 : 0)) * 2 + map) * p.hg_max + h; };

  f32x2 ml[kBatch][2];
  f32x4 o[kBatch][2];
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * kDiffWaves * kRows + rg;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int64_t r = row_of(c < nc ? c : nc - 1, m);  // (past the last: read again, weight 0)
        ml[u][m] = *reinterpret_cast<const f32x2*>(p.part_ml + r * 2);
        o[u][m] = *reinterpret_cast<const f32x4*>(p.part_o32 + r * D + (dl ? 4 * rl : 0));
      }
    }
  };
  constexpr int kStep = kDiffWaves * kRows * kBatch;
  const float lam = p.lambdas[head];
  f32x4 weight = {1.f, 1.f, 1.f, 1.f};
  if (p.norm_weight && dl) weight = *reinterpret_cast<const f32x4*>(p.norm_weight + 4 * rl);
  load(w * kRows);
  float big[2] = {-INFINITY, -INFINITY};
  for (int c = lane; c < nc; c += kWave) {
#pragma unroll
    for (int m = 0; m < 2; ++m) big[m] = fmaxf(big[m], p.part_ml[row_of(c, m) * 2]);
  }
  float ref[2], l[2] = {0.f, 0.f};
  f32x4 acc[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) big[m] = fmaxf(big[m], shfl_xor(big[m], off));
    ref[m] = big[m] == -INFINITY ? 0.f : big[m];
    acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int c0 = w * kRows; c0 < nc; c0 += kStep) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (c0 + u * kDiffWaves * kRows + rg < nc) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float f = __builtin_amdgcn_exp2f(ml[u][m].x - ref[m]);
          l[m] += f * ml[u][m].y;
          acc[m] += f * o[u][m];
        }
      }
    }
    if (c0 + kStep < nc) load(c0 + kStep);
  }
#pragma unroll
  for (int off = kLpr; off < kWave; off <<= 1) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      l[m] += shfl_xor(l[m], off);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] += shfl_xor(acc[m][i], off);
    }
  }
  if (rg == 0 && dl) {
#pragma unroll
    for (int m = 0; m < 2; ++m) *reinterpret_cast<f32x4*>(&sum_lds[w][m][4 * rl]) = acc[m];
  }
  if (lane == 0) {
    l_lds[w][0] = l[0];
    l_lds[w][1] = l[1];
  }
  __syncthreads();
  if (w != 0) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    float lm = 0.f;
    f32x4 om = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kDiffWaves; ++u) {
      lm += l_lds[u][m];
      om += *reinterpret_cast<const f32x4*>(&sum_lds[u][m][dl ? 4 * rl : 0]);
    }
    const float inv = lm > 0.f || lm != lm ? 1.f / lm : 0.f;
    x += om * (m ? -lam * inv : inv);
  }
  float scale = p.out_scale;
  if (p.norm_weight) {
    float ss = rg == 0 && dl ? x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3] : 0.f;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) ss += shfl_xor(ss, off);
    scale *= 1.f / sqrtf(ss * (1.f / D) + p.norm_eps);
  }
  if (rg == 0 && dl) {
    f32x4 y = x * scale;
    if (p.norm_weight) y *= weight;
    *reinterpret_cast<u32x2*>(p.out + (row * (p.num_q_heads / 2) + head) * D + 4 * rl) =
        u32x2{Dt<DT>::pack2(y[0], y[1]), Dt<DT>::pack2(y[2], y[3])};
  }
}

}  // namespace
}  // namespace pal
