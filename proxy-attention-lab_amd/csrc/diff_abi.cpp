// C entry points of differential attention over the paged cache: argument
// validation, workspace sizing and launch.
#include "pal_abi_util.h"

namespace {

bool diff_head_dim_supported(int hd, bool kv8) { return hd == 64 || hd == 128 || (!kv8 && (hd == 32 || hd == 96)); }

// The shapes of both differential attention entry points; returns PAL_OK or an error.
int check_diff_dims(const char* op, int dtype, int kv_dtype, int num_q_heads, int num_kv_heads, int head_dim,
                    int tokens_per_page, int64_t num_pages, int64_t page_table_width) {
  const int st = check_attention_dims(op, dtype, num_q_heads, num_kv_heads, head_dim, tokens_per_page, num_pages,
                                      page_table_width);
  if (st != PAL_OK) return st;
  if (kv_dtype != dtype && kv_dtype != PAL_DTYPE_FP8_E4M3)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] pools must hold the queries' dtype or fp8 (dtype codes %d, %d)", op,
                dtype, kv_dtype);
  if (num_kv_heads % 2 != 0)
    return fail(PAL_ERR_RUNTIME, "[%s] num_kv_heads must be even, two to a pair (%d)", op, num_kv_heads);
  const bool kv8 = kv_dtype == PAL_DTYPE_FP8_E4M3;
  if (!diff_head_dim_supported(head_dim, kv8))
    return fail(PAL_ERR_RUNTIME, "[%s] no %skernel for head_dim %d (supported: %s)", op, kv8 ? "fp8 " : "", head_dim,
                kv8 ? "64, 128" : "32, 64, 96, 128");
  return PAL_OK;
}

// Workspace layout of a differential attention call (256-byte aligned offsets);
// nothing in it needs initial contents.
struct DiffLayout {
  size_t cum, lone, tiles, list, part_ml, part_o, total;
};

DiffLayout diff_layout(int64_t num_rows, int head_dim, int hg_max, int workers) {
  const size_t rows = static_cast<size_t>(workers) * 2 * 2 * hg_max;  // partial rows
  DiffLayout l;
  l.cum = 256;  // behind the header
  l.lone = l.cum + align256(static_cast<size_t>(num_rows + 1) * sizeof(int64_t));
  l.tiles = l.lone + align256(static_cast<size_t>(num_rows) * 4 * sizeof(int32_t));
  // (a run has two rows at least and is cut every 8 or more: no more tiles than half the rows)
  l.list = l.tiles + align256((static_cast<size_t>(num_rows) / 2 + 1) * 2 * sizeof(uint32_t));
  l.part_ml = l.list + align256(static_cast<size_t>(workers) * 4 * sizeof(int64_t));
  l.part_o = l.part_ml + align256(rows * 2 * sizeof(float));
  l.total = l.part_o + align256(rows * 2 * head_dim * sizeof(float));
  return l;
}

int diff_heads_per_segment(int num_q_heads, int num_kv_heads) {
  const int group = num_q_heads / num_kv_heads;
  return group < 8 ? group : 8;
}

size_t diff_workspace_size(int dtype, int kv_dtype, int64_t num_rows, int num_q_heads, int num_kv_heads, int head_dim,
                           int tokens_per_page) {
  int workers = 0;
  if (num_rows <= 0 || num_rows > 0x7fffffffLL ||
      check_diff_dims("paged_differential_attention", dtype, kv_dtype, num_q_heads, num_kv_heads, head_dim,
                      tokens_per_page, 0, 0) != PAL_OK ||
      pal::diff_resident_workers(&workers) != hipSuccess)
    return 0;
  return diff_layout(num_rows, head_dim, diff_heads_per_segment(num_q_heads, num_kv_heads), workers).total;
}

// Rows of sequences: row i of sequence i (decode: no map), or of query_to_seq_map[i].
int diff_call(const char* op, bool mapped, const void* queries, const void* k_pool, const void* v_pool, int kv_dtype,
              const float* k_scales, const float* v_scales, const uint32_t* page_table,
              const int32_t* sequence_lengths, const uint32_t* query_to_seq_map, const int32_t* query_token_offset,
              const float* lambdas, const float* norm_weight, float norm_eps, float out_scale, void* out, int dtype,
              int64_t num_rows, int64_t num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
              int tokens_per_page, int64_t num_pages, int64_t page_table_width, void* workspace,
              size_t workspace_bytes, hipStream_t stream) {
  const int st = check_diff_dims(op, dtype, kv_dtype, num_q_heads, num_kv_heads, head_dim, tokens_per_page, num_pages,
                                 page_table_width);
  if (st != PAL_OK) return st;
  const bool kv8 = kv_dtype == PAL_DTYPE_FP8_E4M3;
  if (kv8 != (k_scales != nullptr) || kv8 != (v_scales != nullptr))
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] k_scales and v_scales go with fp8 pools, both", op);
  if (num_rows < 0 || num_seqs < 0) return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] negative dimension", op);
  if (num_rows > 0x7fffffffLL || num_seqs > 0x7fffffffLL || page_table_width > 0x7fffffffLL / tokens_per_page)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] problem too large for one call", op);
  if (!(norm_eps >= 0.f)) return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] norm_eps must not be negative", op);
  if (num_rows == 0) return ok();
  if (num_pages == 0 || num_seqs == 0) page_table_width = 0;  // no page to read: every row is empty
  if (!queries || (num_seqs > 0 && !sequence_lengths) || !lambdas || !out || (num_pages > 0 && (!k_pool || !v_pool)) ||
      (page_table_width > 0 && !page_table) || (mapped && (!query_to_seq_map || !query_token_offset)))
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] null pointer argument", op);
  if (!aligned16(queries) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(norm_weight) || !aligned16(out))
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] queries, pools, norm_weight and out must be 16-byte aligned", op);
  int workers = 0;
  const hipError_t err = pal::diff_resident_workers(&workers);
  if (err != hipSuccess) return hip_status(err, op);
  const int hg_max = diff_heads_per_segment(num_q_heads, num_kv_heads);
  const DiffLayout lay = diff_layout(num_rows, head_dim, hg_max, workers);
  if (workspace == nullptr || workspace_bytes < lay.total)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] workspace of %zu bytes needed, %zu given", op, lay.total,
                workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] workspace must be 256-byte aligned", op);
  pal::DiffParams p{};
  p.q = static_cast<const uint16_t*>(queries);
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.k_scales = k_scales;
  p.v_scales = v_scales;
  p.page_table = page_table;
  p.seq_lens = sequence_lengths;
  p.out = static_cast<uint16_t*>(out);
  p.q2seq = mapped ? query_to_seq_map : nullptr;
  p.q_offset = mapped ? query_token_offset : nullptr;
  p.num_pt_rows = num_seqs;
  p.num_seqs = num_rows;
  p.num_pages = num_pages;
  p.page_table_width = page_table_width;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads / 2;
  p.group = num_q_heads / num_kv_heads;
  p.head_chunks = (p.group + 7) / 8;
  p.hg_max = hg_max;
  p.num_workers = workers;
  p.tile_chunks = (p.group + 15) / 16;
  p.tile_heads = (p.group + p.tile_chunks - 1) / p.tile_chunks;
  p.tile_magic = (65536u + p.tile_heads - 1) / p.tile_heads;
  p.tile_rows = 128 / p.tile_heads;
  {  // 2^l / tile_rows rounded up, exact for x < 2^31 (tile_rows is 8 or more)
    int log2 = 3;
    while (2 << log2 <= p.tile_rows) ++log2;
    const bool pow2 = 1 << log2 == p.tile_rows;
    p.rows_shift = static_cast<uint32_t>(pow2 ? log2 - 1 : log2);
    p.rows_magic = pow2 ? 1u << 31 : static_cast<uint32_t>((1ull << (32 + log2)) / p.tile_rows + 1);
  }
  if ((num_rows / 2 + 1) * p.num_kv_heads * p.tile_chunks > 0x7fffffffLL)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] problem too large for one call", op);
  p.scale_log2 = scale_log2_for(head_dim);
  char* ws = static_cast<char*>(workspace);
  p.hdr = reinterpret_cast<int64_t*>(ws);
  p.claim = reinterpret_cast<uint32_t*>(ws + 128);
  p.cum = reinterpret_cast<int64_t*>(ws + lay.cum);
  p.split_list = reinterpret_cast<int64_t*>(ws + lay.list);
  p.list_cap = workers;
  p.lone = reinterpret_cast<int32_t*>(ws + lay.lone);
  p.tiles = reinterpret_cast<uint32_t*>(ws + lay.tiles);
  p.part_ml = reinterpret_cast<float*>(ws + lay.part_ml);
  p.part_o32 = reinterpret_cast<float*>(ws + lay.part_o);
  p.lambdas = lambdas;
  p.norm_weight = norm_weight;
  p.norm_eps = norm_eps;
  p.out_scale = out_scale;
  PAL_LOG("%s rows=%lld seqs=%lld Hq=%d Hkv=%d HD=%d TPP=%d dtype=%d kv=%d norm=%d stream=%p", op,
          static_cast<long long>(num_rows), static_cast<long long>(num_seqs), num_q_heads, num_kv_heads, head_dim,
          tokens_per_page, dtype, kv_dtype, norm_weight ? 1 : 0, static_cast<void*>(stream));
  return hip_status(pal::launch_diff(p, dtype, head_dim, tokens_per_page, stream), op);
}

}  // namespace

extern "C" {

size_t pal_paged_differential_attention_workspace_size(int dtype, int kv_dtype, int64_t num_query_rows,
                                                       int num_q_heads, int num_kv_heads, int head_dim,
                                                       int tokens_per_page) {
  return diff_workspace_size(dtype, kv_dtype, num_query_rows, num_q_heads, num_kv_heads, head_dim, tokens_per_page);
}

int pal_paged_differential_attention_decode(const void* queries, const void* k_pool, const void* v_pool, int kv_dtype,
                                            const float* k_scales, const float* v_scales, const uint32_t* page_table,
                                            const int32_t* sequence_lengths, const float* lambdas,
                                            const float* norm_weight, float norm_eps, float out_scale, void* out,
                                            int dtype, int64_t num_query_rows, int64_t num_seqs, int num_q_heads,
                                            int num_kv_heads, int head_dim, int tokens_per_page, int64_t num_pages,
                                            int64_t page_table_width, void* workspace, size_t workspace_bytes,
                                            void* stream) {
  const char* op = "paged_differential_attention_decode";
  if (num_query_rows < num_seqs)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] %lld query rows for %lld sequences", op,
                static_cast<long long>(num_query_rows), static_cast<long long>(num_seqs));
  return diff_call(op, false, queries, k_pool, v_pool, kv_dtype, k_scales, v_scales, page_table, sequence_lengths,
                   nullptr, nullptr, lambdas, norm_weight, norm_eps, out_scale, out, dtype, num_seqs, num_seqs,
                   num_q_heads, num_kv_heads, head_dim, tokens_per_page, num_pages, page_table_width, workspace,
                   workspace_bytes, static_cast<hipStream_t>(stream));
}

int pal_paged_differential_attention(const void* queries, const void* k_pool, const void* v_pool, int kv_dtype,
                                     const float* k_scales, const float* v_scales, const uint32_t* page_table,
                                     const int32_t* sequence_lengths, const uint32_t* query_to_seq_map,
                                     const int32_t* query_token_offset, const float* lambdas,
                                     const float* norm_weight, float norm_eps, float out_scale, void* out, int dtype,
                                     int64_t num_query_rows, int64_t num_seqs, int num_q_heads, int num_kv_heads,
                                     int head_dim, int tokens_per_page, int64_t num_pages, int64_t page_table_width,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  return diff_call("paged_differential_attention", true, queries, k_pool, v_pool, kv_dtype, k_scales, v_scales,
                   page_table, sequence_lengths, query_to_seq_map, query_token_offset, lambdas, norm_weight, norm_eps,
                   out_scale, out, dtype, num_query_rows, num_seqs, num_q_heads, num_kv_heads, head_dim,
                   tokens_per_page, num_pages, page_table_width, workspace, workspace_bytes,
                   static_cast<hipStream_t>(stream));
}

}  // extern "C"
