// Attention over the paged K/V cache: argument checks, the choice of kernel
// and the launches.
#include "attn_rows.cuh"

namespace d3 {

// Rows of a cache buffer ([rows][D], one row per token and head) in boxes of
// box_rows x 128 bytes, 128-byte swizzle; rows outside read as zeros.
static int make_rows_map(CUtensorMap* m, const void* base, int dtype, uint64_t D, uint64_t rows,
                         uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(D3_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  const uint32_t es = dtype == D3_E4M3 ? 1 : 2;
  cuuint64_t dims[2] = {D, rows};
  cuuint64_t strides[1] = {D * es};
  cuuint32_t box[2] = {128 / es, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType t = dtype == D3_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : dtype == D3_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  CUresult r = fn(m, t, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(D3_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return D3_OK;
}

static int check_attention(const d3_attention* a, const d3_kv_cache* c) {
  D3_CHECK_ARG(a, "d3_paged_attention: null arguments");
  int rc = check_kv_cache(c, "d3_paged_attention");
  if (rc) return rc;
  D3_CHECK_ARG(a->dtype == D3_BF16 || a->dtype == D3_F16, "d3_paged_attention: q must be bf16 or fp16");
  D3_CHECK_ARG(c->dtype == D3_E4M3 || c->dtype == a->dtype,
               "d3_paged_attention: a 16-bit cache takes queries of its own type");
  D3_CHECK_ARG(a->batch >= 0 && a->tokens >= 0 && a->heads >= 1 && a->table_pages >= 0 && a->max_q >= 1 &&
                   a->max_kv >= 0 && a->table_stride >= 0,
               "d3_paged_attention: sizes out of range");
  D3_CHECK_ARG(a->heads % c->kv_heads == 0, "d3_paged_attention: %d heads over %d KV heads", (int)a->heads,
               (int)c->kv_heads);
  if (a->heads / c->kv_heads > 128)
    return fail(D3_ERR_UNSUPPORTED, "d3_paged_attention: %d query heads a KV head (128 at most)",
                (int)(a->heads / c->kv_heads));
  if ((long long)a->tokens * (a->heads / c->kv_heads) >= (1LL << 30) ||
      (long long)a->table_pages * c->page_size >= (1LL << 30) || (long long)a->batch * c->kv_heads >= (1LL << 24))
    return fail(D3_ERR_TOO_LARGE, "d3_paged_attention: tokens, table or batch too large");
  D3_CHECK_ARG(a->scale == a->scale, "d3_paged_attention: scale is NaN");
  return D3_OK;
}

constexpr int kJoinGroups = 4;   // row groups of a sequence's KV head with a join CTA of their own

template <typename T, int D, bool E4, int NT>
static int launch_rows(AttnParams p, const d3_attention* a, const d3_kv_cache* c, cudaStream_t st) {
  using C = RowsCfg<T, D, E4, NT>;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    D3_CUDA_TRY(cudaFuncSetAttribute(attn_rows_kernel<T, D, E4, NT>,
                                     cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM),
                "attention smem attribute");
    attr_set[dev] = true;
  }
  const uint32_t box = c->page_size < C::KEYS ? c->page_size : C::KEYS;
  const uint64_t rows = (uint64_t)c->pages * c->kv_heads * c->page_size;
  CUtensorMap tk, tv;
  int rc;
  if ((rc = make_rows_map(&tk, c->k, c->dtype, D, rows, box))) return rc;
  if ((rc = make_rows_map(&tv, c->v, c->dtype, D, rows, box))) return rc;
  const long long groups = ((long long)a->max_q * p.group + C::ROWS - 1) / C::ROWS;
  const long long tiles = ((long long)a->max_kv + C::KEYS - 1) / C::KEYS;
  const long long most = (tiles < 1 ? 1 : tiles) * groups * a->batch * c->kv_heads;
  const int parts = (int)(most < num_sms() ? most : num_sms());
  D3_CUDA_TRY(launch_k(attn_rows_kernel<T, D, E4, NT>, dim3(parts), dim3(C::THREADS), C::SMEM, st,
                       pdl_enabled(), tk, tv, p),
              "attn_rows_kernel launch");
  const int jg = (int)(groups < kJoinGroups ? groups : kJoinGroups);
  D3_CUDA_TRY(launch_k(attn_rows_join_kernel<T, D>, dim3((unsigned)(a->batch * c->kv_heads * jg)), dim3(128), 0,
                       st, pdl_enabled(), p, (int)C::KEYS, (int)C::ROWS, parts, jg),
              "attn_rows_join_kernel launch");
  return D3_OK;
}

template <typename T, int D, bool E4>
static int launch_rows_nt(const AttnParams& p, const d3_attention* a, const d3_kv_cache* c, cudaStream_t st) {
  return a->max_q * p.group <= 8 ? launch_rows<T, D, E4, 1>(p, a, c, st) : launch_rows<T, D, E4, 2>(p, a, c, st);
}

}  // namespace d3

using namespace d3;

extern "C" {

size_t d3_paged_attention_workspace_size(const d3_attention* a, const d3_kv_cache* c) {
  if (check_attention(a, c)) return 0;
  // two places per CTA of the row kernel: 16 rows of sums, maxima and sums
  return (size_t)num_sms() * 2 * 16 * ((size_t)c->head_dim + 2) * 4 + 256;
}

int d3_paged_attention(const d3_attention* a, const d3_kv_cache* c, int32_t* err_word, void* workspace,
                       size_t workspace_bytes, d3_stream_t stream) {
  int rc = check_attention(a, c);
  if (rc) return rc;
  if (a->batch == 0 || a->tokens == 0) return D3_OK;
  D3_CHECK_ARG(a->q && a->out && a->kv_lens && (a->page_table || a->table_pages == 0) && err_word,
               "d3_paged_attention: null pointer");
  if (!aligned16(a->q) || !aligned16(a->out) || a->q_token % 8 || a->q_head % 8 || a->out_token % 8 || a->out_head % 8)
    return fail(D3_ERR_MISALIGNED, "d3_paged_attention: rows must start on 16-byte boundaries");
  D3_CHECK_ARG(a->cu_q || a->tokens >= a->batch, "d3_paged_attention: without cu_q every sequence has a row");
  if (!workspace || workspace_bytes < d3_paged_attention_workspace_size(a, c))
    return fail(D3_ERR_WORKSPACE, "d3_paged_attention: workspace of %zu bytes needed",
                d3_paged_attention_workspace_size(a, c));
  if (!aligned16(workspace)) return fail(D3_ERR_MISALIGNED, "d3_paged_attention: workspace not 16-byte aligned");
  AttnParams p{};
  p.q = a->q;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.out = a->out;
  p.out_token = a->out_token;
  p.out_head = a->out_head;
  p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.table_pages = a->table_pages;
  p.kv_lens = a->kv_lens;
  p.cu_q = a->cu_q;
  p.batch = a->batch;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = c->kv_heads;
  p.group = a->heads / c->kv_heads;
  p.page_size = c->page_size;
  p.page_shift = __builtin_ctz((unsigned)c->page_size);
  p.pages = c->pages;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  p.scale_log2 = a->scale * 1.44269504088896340736f;
  p.min_rows = 0;
  p.max_rows = 0x7fffffff;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = p.ws_o + (size_t)num_sms() * 2 * 16 * c->head_dim;
  p.err = err_word;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool e4 = c->dtype == D3_E4M3;
  if (a->dtype == D3_BF16) {
    if (c->head_dim == 128)
      return e4 ? launch_rows_nt<__nv_bfloat16, 128, true>(p, a, c, st) : launch_rows_nt<__nv_bfloat16, 128, false>(p, a, c, st);
    return e4 ? launch_rows_nt<__nv_bfloat16, 256, true>(p, a, c, st) : launch_rows_nt<__nv_bfloat16, 256, false>(p, a, c, st);
  }
  if (c->head_dim == 128)
    return e4 ? launch_rows_nt<__half, 128, true>(p, a, c, st) : launch_rows_nt<__half, 128, false>(p, a, c, st);
  return e4 ? launch_rows_nt<__half, 256, true>(p, a, c, st) : launch_rows_nt<__half, 256, false>(p, a, c, st);
}

}  // extern "C"
