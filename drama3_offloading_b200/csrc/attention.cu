// Attention over the paged K/V cache: argument checks, the choice of kernel
// and the launches.
#include "attn_chunk.cuh"

namespace d3 {

// A tensor map, with the 128-byte swizzle unless told otherwise; what lies
// outside reads as zeros.
static int make_map(CUtensorMap* m, const void* base, int dtype, int rank, const uint64_t* dims,
                    const uint64_t* strides, const uint32_t* box, bool swizzle = true) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(D3_ERR_CUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  cuuint64_t d[4], s[3];
  cuuint32_t x[4], e[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    x[i] = box[i];
    if (i) s[i - 1] = strides[i - 1];
  }
  const CUtensorMapDataType t = dtype == D3_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : dtype == D3_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  CUresult r = fn(m, t, rank, const_cast<void*>(base), d, s, x, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(D3_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return D3_OK;
}

// A cache buffer as planes [pages * kv_heads][page_size][D], the dims in
// columns of 128 bytes, swizzled -- or, for codes that are to be widened, in
// one, unswizzled.  Rows before or behind a page are outside the map.
static int make_pages_map(CUtensorMap* m, const void* base, const d3_kv_cache* c, bool swizzle, uint32_t box_dims,
                          uint32_t box_rows, uint32_t box_cols) {
  const uint64_t D = c->head_dim, es = c->dtype == D3_E4M3 ? 1 : 2, col = swizzle ? 128 / es : D;
  const uint64_t dims[4] = {col, (uint64_t)c->page_size, D / col, (uint64_t)c->pages * c->kv_heads};
  const uint64_t strides[3] = {D * es, col * es, c->page_size * D * es};
  const uint32_t box[4] = {box_dims, box_rows, box_cols, 1};
  return make_map(m, base, c->dtype, 4, dims, strides, box, swizzle);
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
  D3_CHECK_ARG(a->scale > 0.f && a->scale < INFINITY, "d3_paged_attention: scale must be positive");
  return D3_OK;
}

// Up to this many rows of a KV head (new tokens x query heads that share it) a
// sequence goes through the row kernel.  Above it the row kernel would read
// the keys once per 16 rows; the 256-row pairs of the chunk kernel read them
// once and, although most of their rows may be empty, keep up with HBM.
constexpr int kRowsMost = 16;

// SMs that the kernels' parts are counted for: a part of either kernel has a
// thread of a joining block.
static int part_sms() {
  const int n = num_sms();
  return n < kJoinThreads * 2 / 3 ? n : kJoinThreads * 2 / 3;
}

struct Workspace {         // byte offsets
  size_t rows_o, rows_ml, rows_desc, chunk_o, chunk_ml, chunk_desc, total;
};
static Workspace plan_workspace(const d3_attention* a, const d3_kv_cache* c) {
  Workspace w{};
  const size_t D = c->head_dim, sms = part_sms(), pairs = sms / 2;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = (at + n + 255) / 256 * 256;
    return o;
  };
  w.rows_o = take(sms * 2 * kRowsMost * D * 4);
  w.rows_ml = take(sms * 2 * kRowsMost * 8);
  w.rows_desc = take(sms * 32);
  if ((long long)a->max_q * (a->heads / c->kv_heads) > kRowsMost) {
    w.chunk_o = take(pairs * 2 * 256 * D * 4);
    w.chunk_ml = take(pairs * 2 * 256 * 8);
    w.chunk_desc = take(pairs * 32);
  }
  w.total = at;
  return w;
}

template <typename K>
static int set_smem(K kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    D3_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
                "attention smem attribute");
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return D3_OK;
}

template <typename T, int D, bool E4, int NT>
static int launch_rows(const AttnParams& p, const d3_attention* a, const d3_kv_cache* c, int* parts_out, cudaStream_t st) {
  using C = RowsCfg<T, D, E4, NT>;
  static bool done[64] = {false};
  int rc;
  if ((rc = set_smem(attn_rows_kernel<T, D, E4, NT>, C::SMEM, done))) return rc;
  const uint32_t box = c->page_size < C::KEYS ? c->page_size : C::KEYS;
  CUtensorMap tk, tv;
  if ((rc = make_pages_map(&tk, c->k, c, true, 128 / C::ES, box, C::COLS))) return rc;
  if ((rc = make_pages_map(&tv, c->v, c, true, 128 / C::ES, box, C::COLS))) return rc;
  const long long groups = ((long long)a->max_q * p.group + C::ROWS - 1) / C::ROWS;
  const long long tiles = ((long long)a->max_kv + C::KEYS - 1) / C::KEYS;
  // the kernel counts the list in 31 bits; what it reads may be larger than max_q and max_kv say
  if (((long long)a->tokens * p.group / C::ROWS + a->batch) * c->kv_heads *
          ((long long)a->table_pages * c->page_size / C::KEYS + 1 + kPieceUnits) >= kListMost)
    return fail(D3_ERR_TOO_LARGE, "d3_paged_attention: too many key tiles");
  const long long most = (tiles < 1 ? 1 : tiles) * groups * a->batch * c->kv_heads;
  const int parts = (int)(most < part_sms() ? most : part_sms());
  D3_CUDA_TRY(launch_k(attn_rows_kernel<T, D, E4, NT>, dim3(parts), dim3(C::THREADS), C::SMEM, st,
                       pdl_enabled(), tk, tv, p),
              "attn_rows_kernel launch");
  *parts_out = parts;
  return D3_OK;
}

template <typename T, int D, bool E4>
static int launch_chunk(const AttnParams& p, const d3_attention* a, const d3_kv_cache* c, const ChunkWs& ws,
                        int* pairs_out, cudaStream_t st) {
  using C = ChunkCfg<T, D, E4>;
  static bool done[64] = {false};
  int rc;
  if ((rc = set_smem(attn_chunk_kernel<T, D, E4>, C::SMEM, done))) return rc;
  const int tpc = 128 / p.group;
  CUtensorMap tq, tk, tv;
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)a->heads, (uint64_t)a->tokens};
  const uint64_t strides[2] = {(uint64_t)a->q_head * 2, (uint64_t)a->q_token * 2};
  const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)tpc};
  if ((rc = make_map(&tq, a->q, a->dtype, 3, dims, strides, box))) return rc;
  const uint32_t krows = c->page_size < 64 ? c->page_size : 64;
  if ((rc = make_pages_map(&tk, c->k, c, !E4, E4 ? D : 64, krows, !E4 && krows == 64 ? D / 64 : 1))) return rc;
  if ((rc = make_pages_map(&tv, c->v, c, !E4, E4 ? D / 2 : 64, c->page_size, E4 ? 1 : D / 128))) return rc;
  // row tiles at most: every sequence may have one that is not full
  const long long tiles = a->tokens / (2 * tpc) + a->batch;
  const long long blocks = ((long long)a->max_kv + kBlockKeys - 1) / kBlockKeys;
  const long long most = (blocks < 1 ? 1 : blocks) * tiles * c->kv_heads;
  // the kernel counts the list in 31 bits; the lengths it reads may be larger than max_kv says
  if (((long long)a->table_pages * c->page_size / kBlockKeys + 1 + kTileUnits<D>) * tiles * c->kv_heads >= kListMost)
    return fail(D3_ERR_TOO_LARGE, "d3_paged_attention: too many key blocks");
  const int pairs = (int)(most < part_sms() / 2 ? most : part_sms() / 2);
  D3_CUDA_TRY(launch_k(attn_chunk_kernel<T, D, E4>, dim3(2 * pairs), dim3(C::THREADS), C::SMEM, st, pdl_enabled(),
                       tq, tk, tv, p, ws),
              "attn_chunk_kernel launch");
  *pairs_out = pairs;
  return D3_OK;
}

// Which kernels run.  One launch pair for all sequences where max_q says that
// all are short, or where tokens == batch * max_q says that none is (a shorter
// one is still right there); otherwise each kernel takes its own.
template <typename T, int D, bool E4>
static int launch_attention(AttnParams p, const d3_attention* a, const d3_kv_cache* c, const ChunkWs& ws,
                            cudaStream_t st) {
  const long long rows = (long long)a->max_q * p.group;
  int rc = D3_OK, parts = 0, pairs = 0, rows_per = 8;
  if (rows <= kRowsMost) {
    rows_per = rows <= 8 ? 8 : 16;
    rc = rows_per == 8 ? launch_rows<T, D, E4, 1>(p, a, c, &parts, st) : launch_rows<T, D, E4, 2>(p, a, c, &parts, st);
  } else {
    if ((long long)a->batch * a->max_q != a->tokens && p.group <= kRowsMost) {
      // mostly single tokens among chunks: eight rows where a token has no more
      // (sixteen cost the row kernel twice the products)
      AttnParams few = p;
      few.max_rows = rows_per = p.group <= 8 ? 8 : kRowsMost;
      d3_attention one = *a;
      one.max_q = few.max_rows / p.group;
      if ((rc = rows_per == 8 ? launch_rows<T, D, E4, 1>(few, &one, c, &parts, st)
                              : launch_rows<T, D, E4, 2>(few, &one, c, &parts, st)))
        return rc;
      p.min_rows = few.max_rows + 1;
      p.beside = 1;
    }
    rc = launch_chunk<T, D, E4>(p, a, c, ws, &pairs, st);
  }
  if (rc) return rc;
  const int items = parts * rows_per + pairs * (256 / kJoinRows), most = kJoinBlocks * num_sms();
  const dim3 grid = pairs ? dim3(items < most ? items : most) : dim3(parts, rows_per);
  D3_CUDA_TRY(launch_k(attn_join_kernel<T, D>, grid, dim3(kJoinThreads), 0, st,
                       pdl_enabled(), p, rows_per, parts, parts + pairs, ws),
              "attn_join_kernel launch");
  return D3_OK;
}

}  // namespace d3

using namespace d3;

extern "C" {

size_t d3_paged_attention_workspace_size(const d3_attention* a, const d3_kv_cache* c) {
  if (check_attention(a, c)) return 0;
  return plan_workspace(a, c).total;
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
  const Workspace w = plan_workspace(a, c);
  if (!workspace || workspace_bytes < w.total)
    return fail(D3_ERR_WORKSPACE, "d3_paged_attention: workspace of %zu bytes needed", w.total);
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
  char* base = static_cast<char*>(workspace);
  p.ws_o = reinterpret_cast<float*>(base + w.rows_o);
  p.ws_ml = reinterpret_cast<float*>(base + w.rows_ml);
  p.ws_desc = reinterpret_cast<int4*>(base + w.rows_desc);
  const ChunkWs ws{reinterpret_cast<float*>(base + w.chunk_o), reinterpret_cast<float*>(base + w.chunk_ml),
                   reinterpret_cast<int4*>(base + w.chunk_desc)};
  p.k_codes = c->k;
  p.v_codes = c->v;
  p.err = err_word;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool e4 = c->dtype == D3_E4M3;
  if (a->dtype == D3_BF16) {
    if (c->head_dim == 128)
      return e4 ? launch_attention<__nv_bfloat16, 128, true>(p, a, c, ws, st) : launch_attention<__nv_bfloat16, 128, false>(p, a, c, ws, st);
    return e4 ? launch_attention<__nv_bfloat16, 256, true>(p, a, c, ws, st) : launch_attention<__nv_bfloat16, 256, false>(p, a, c, ws, st);
  }
  if (c->head_dim == 128)
    return e4 ? launch_attention<__half, 128, true>(p, a, c, ws, st) : launch_attention<__half, 128, false>(p, a, c, ws, st);
  return e4 ? launch_attention<__half, 256, true>(p, a, c, ws, st) : launch_attention<__half, 256, false>(p, a, c, ws, st);
}

}  // extern "C"
