// The paged K/V cache and what fills it: quantising write, read back, and the
// norm and rotation of queries and keys, alone or in one pass with the write.
//
//   norm      y_i = x_i / sqrt(mean(x^2) + eps) * (w_i + offset), one head at
//             a time, the mean in fp32.
//   rotation  the first R dims of y in pairs (i, i + R/2), or (2i, 2i + 1),
//             turned by pos * inv_freq[i].  The angle is taken in turns in
//             fp64 and only its fraction goes on in fp32: at position 10^6 an
//             fp32 angle would be 0.03 rad off.
//   cached    16-bit rows as they are; e4m3 rows as codes e4m3(y / s) with one
//             fp32 s = max|y| / 448 per (token, head), s = 1 for a row of
//             zeros.  Both divisions are IEEE ones, so the codes are those of
//             the formula bit for bit.  K is quantised from the fp32 result of
//             the rotation: one rounding, not two.
//
// All of it is bound by HBM for large batches (every element is read once and
// written once) and by launch latency for a decode token.  A head row is held
// by D/8 lanes, 16 bytes each, so its sums are lane shuffles and the rotation
// of halves is a shuffle by R/16 lanes; nothing goes through shared memory but
// the sines of a token, which all of its heads use.
#include "kv_common.cuh"

namespace d3 {

int check_kv_cache(const d3_kv_cache* c, const char* who) {
  D3_CHECK_ARG(c && c->k && c->v, "%s: null cache", who);
  D3_CHECK_ARG(c->dtype == D3_BF16 || c->dtype == D3_F16 || c->dtype == D3_E4M3,
               "%s: cache dtype %d", who, (int)c->dtype);
  D3_CHECK_ARG(c->pages >= 1 && c->kv_heads >= 1, "%s: pages and kv_heads must be >= 1", who);
  if (c->head_dim != 128 && c->head_dim != 256)
    return fail(D3_ERR_UNSUPPORTED, "%s: head_dim %d (128 or 256)", who, (int)c->head_dim);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(D3_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64 or 128)", who,
                (int)c->page_size);
  // rows of the cache are counted in 31 bits (a tensor map's coordinate)
  if ((long long)c->pages * c->kv_heads * c->page_size >= (1LL << 31))
    return fail(D3_ERR_TOO_LARGE, "%s: pages * kv_heads * page_size must be below 2^31", who);
  if (!aligned16(c->k) || !aligned16(c->v))
    return fail(D3_ERR_MISALIGNED, "%s: cache not 16-byte aligned", who);
  D3_CHECK_ARG(c->dtype != D3_E4M3 || (c->k_scale && c->v_scale),
               "%s: an e4m3 cache needs its scales", who);
  if (c->dtype == D3_E4M3 && (!aligned16(c->k_scale) || !aligned16(c->v_scale)))
    return fail(D3_ERR_MISALIGNED, "%s: scales not 16-byte aligned", who);
  return D3_OK;
}

struct RowsIn {           // [tokens][heads][D], strides in elements
  const void* p;
  long long token, head;
};

struct FillParams {
  RowsIn q, k, v;
  void *q_out, *k_out;    // k_out: NULL when K goes into the cache
  long long q_out_token, q_out_head, k_out_token, k_out_head;
  const void *q_w, *k_w;
  const void* positions;
  const double* inv_freq;
  const void* slots;
  int pos_bytes, slot_bytes, tokens, heads, kv_heads, half, interleaved;
  int tokens_per_cta;
  float eps, w_offset;
  d3_kv_cache cache;      // k == NULL: no cache
};

constexpr int kFillThreads = 256;
constexpr int kMaxHalf = 128;          // rotary pairs of the widest head
constexpr int kMaxTokensPerCta = 4;

// A group of D/8 lanes holds one row; NORM: norm and rotation of q and k rows
// (otherwise there are no q rows and K goes in as it is).
template <typename T, int D, bool NORM>
__global__ void __launch_bounds__(kFillThreads) kv_fill_kernel(const __grid_constant__ FillParams p) {
  constexpr int L = D / 8;                          // lanes of a row
  __shared__ float s_cos[kMaxTokensPerCta][kMaxHalf], s_sin[kMaxTokensPerCta][kMaxHalf];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  constexpr int GROUPS = kFillThreads / L;
  const int t0 = blockIdx.x * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.tokens - t0);
  pdl_trigger();
  pdl_wait();
  if (NORM) {
    for (int i = threadIdx.x; i < nt * p.half; i += kFillThreads) {
      const int t = i / p.half, j = i - t * p.half;
      const double turns = (double)load_index(p.positions, p.pos_bytes, t0 + t) * p.inv_freq[j] *
                           0.15915494309189533577;  // 1 / (2 pi)
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      s_cos[t][j] = c;
      s_sin[t][j] = s;
    }
    __syncthreads();
  }
  const bool cached = p.cache.k != nullptr;
  const int rows = p.heads + (cached ? 2 : 1) * p.kv_heads;   // q, k and, into a cache, v
  // every lane of a warp takes the same number of turns: the shuffles are whole
  for (int r0 = 0; r0 < nt * rows; r0 += GROUPS) {
    const int r = r0 + grp;
    const bool live = r < nt * rows;
    const int t = live ? r / rows : 0, h = live ? r - t * rows : 0;
    const int kind = h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;
    const int head = kind == 0 ? h : kind == 1 ? h - p.heads : h - p.heads - p.kv_heads;
    const RowsIn& in = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const long long tok = t0 + t;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live)
      raw = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(in.p) + tok * in.token +
                                                  head * in.head + lane * 8));
    float x[8];
    unpack8<T>(raw, x);
    if (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (kind < 2) {
        const float inv = 1.f / sqrtf(ss * (1.f / D) + p.eps);
        float w[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(
                       static_cast<const T*>(kind == 0 ? p.q_w : p.k_w) + lane * 8), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * (w[i] + p.w_offset);
      }
      const float *cs = s_cos[t], *sn = s_sin[t];
      if (p.interleaved) {
        if (kind < 2 && lane * 4 < p.half) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float c = cs[lane * 4 + i], s = sn[lane * 4 + i];
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = a * c - b * s;
            x[2 * i + 1] = b * c + a * s;
          }
        }
      } else {
        // lanes [0, R/16) hold the first halves, the next R/16 the second
        const int n = p.half / 8;
        const bool first = lane < n;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          y[i] = __shfl_sync(0xffffffffu, x[i], first ? lane + n : lane - n, L);
        if (kind < 2 && lane < 2 * n) {
          const int j = (first ? lane : lane - n) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float c = cs[j + i], s = sn[j + i];
            x[i] = first ? x[i] * c - y[i] * s : x[i] * c + y[i] * s;
          }
        }
      }
    }
    float amax = 0.f;
    if (p.cache.dtype == D3_E4M3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1)
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (!live) continue;
    if (kind == 0) {
      *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + tok * p.q_out_token +
                                head * p.q_out_head + lane * 8) = pack8<T>(x);
      continue;
    }
    if (!cached) {
      *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + tok * p.k_out_token +
                                head * p.k_out_head + lane * 8) = pack8<T>(x);
      continue;
    }
    const long long slot = load_index(p.slots, p.slot_bytes, tok);
    if (slot < 0 || slot >= (long long)p.cache.pages * p.cache.page_size) continue;
    const long long page = slot / p.cache.page_size, off = slot - page * p.cache.page_size;
    const long long row = (page * p.cache.kv_heads + head) * p.cache.page_size + off;
    void* base = kind == 1 ? p.cache.k : p.cache.v;
    if (p.cache.dtype == D3_E4M3) {
      const float s = amax > 0.f ? amax / kE4m3Max : 1.f;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = e4m3x2(x[2 * i] / s, x[2 * i + 1] / s);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + row * D + lane * 8) =
          make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      if (lane == 0) (kind == 1 ? p.cache.k_scale : p.cache.v_scale)[row] = s;
    } else {
      *reinterpret_cast<uint4*>(static_cast<T*>(base) + row * D + lane * 8) = pack8<T>(x);
    }
  }
}

struct ReadParams {
  const void* slots;
  int slot_bytes, tokens;
  void *k_out, *v_out;    // [tokens][kv_heads][D], contiguous
  d3_kv_cache cache;
};

constexpr int kReadRows = 2;   // rows a lane group has in flight

// Rows of the cache back in 16 bits: T(code * s), or the row as it is.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int L = D / 8, GROUPS = 256 / L;
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  pdl_trigger();
  pdl_wait();
  const long long per = 2LL * p.cache.kv_heads, rows = p.tokens * per;
  const long long r0 = (long long)blockIdx.x * (GROUPS * kReadRows) + grp;
  long long at[kReadRows];
  const void* src[kReadRows];
  bool live[kReadRows], have[kReadRows];
  uint4 raw[kReadRows];
  float sc[kReadRows];
  T* out[kReadRows];
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const long long r = r0 + i * GROUPS;
    live[i] = r < rows;
    have[i] = false;
    raw[i] = make_uint4(0, 0, 0, 0);
    sc[i] = 1.f;
    if (!live[i]) continue;
    const long long t = r / per;
    const int h2 = (int)(r - t * per), h = h2 >> 1;
    const bool is_k = (h2 & 1) == 0;
    out[i] = static_cast<T*>(is_k ? p.k_out : p.v_out) + (t * p.cache.kv_heads + h) * D + lane * 8;
    const long long slot = load_index(p.slots, p.slot_bytes, t);
    have[i] = slot >= 0 && slot < (long long)p.cache.pages * p.cache.page_size;
    if (!have[i]) continue;
    const long long page = slot / p.cache.page_size, off = slot - page * p.cache.page_size;
    at[i] = (page * p.cache.kv_heads + h) * p.cache.page_size + off;
    src[i] = is_k ? p.cache.k : p.cache.v;
    if (p.cache.dtype == D3_E4M3) {
      const uint2 c = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(src[i]) +
                                                            at[i] * D + lane * 8));
      raw[i].x = c.x;
      raw[i].y = c.y;
      sc[i] = __ldcg((is_k ? p.cache.k_scale : p.cache.v_scale) + at[i]);
    } else {
      raw[i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src[i]) +
                                                     at[i] * D + lane * 8));
    }
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    if (!live[i]) continue;
    uint4 o = raw[i];
    float x[8];
    if (p.cache.dtype == D3_E4M3) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = j < 2 ? raw[i].x : raw[i].y;
        const float2 f = e4m3x2_to_f2((uint16_t)(j & 1 ? w >> 16 : w));
        x[2 * j] = f.x * sc[i];
        x[2 * j + 1] = f.y * sc[i];
      }
      o = have[i] ? pack8<T>(x) : make_uint4(0, 0, 0, 0);
    }
    *reinterpret_cast<uint4*>(out[i]) = o;
  }
}

// ---------------------------------------------------------------- host

// Tokens a CTA takes: one for small batches (as many CTAs as tokens, so that
// a decode batch spreads over the SMs), four once there are enough tokens for
// every SM to hold several CTAs all the same.
static int tokens_per_cta(int tokens) { return tokens >= 8 * num_sms() ? kMaxTokensPerCta : 1; }

template <typename T>
static int launch_fill(const FillParams& p, int D, bool norm, cudaStream_t st) {
  const dim3 grid((unsigned)((p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta));
  void (*k)(FillParams) = D == 128 ? (norm ? kv_fill_kernel<T, 128, true> : kv_fill_kernel<T, 128, false>)
                                   : (norm ? kv_fill_kernel<T, 256, true> : kv_fill_kernel<T, 256, false>);
  D3_CUDA_TRY(launch_k(k, grid, dim3(kFillThreads), 0, st, pdl_enabled(), p), "kv_fill_kernel launch");
  return D3_OK;
}

static int check_rows(const void* p, int64_t token, int64_t head, const char* what) {
  D3_CHECK_ARG(p, "%s: null pointer", what);
  if (!aligned16(p) || token % 8 || head % 8)
    return fail(D3_ERR_MISALIGNED, "%s: rows must start on 16-byte boundaries", what);
  return D3_OK;
}

}  // namespace d3

using namespace d3;

extern "C" {

int d3_kv_write(const d3_kv_cache* cache, const void* k, int64_t k_token, int64_t k_head,
                const void* v, int64_t v_token, int64_t v_head, int32_t dtype, int32_t tokens,
                const void* slots, int32_t slot_bytes, d3_stream_t stream) {
  int rc = check_kv_cache(cache, "d3_kv_write");
  if (rc) return rc;
  D3_CHECK_ARG(dtype == D3_BF16 || dtype == D3_F16, "d3_kv_write: rows must be bf16 or fp16");
  D3_CHECK_ARG(cache->dtype == D3_E4M3 || cache->dtype == dtype,
               "d3_kv_write: a 16-bit cache takes rows of its own type");
  D3_CHECK_ARG(slot_bytes == 4 || slot_bytes == 8, "slot_bytes must be 4 or 8");
  D3_CHECK_ARG(tokens >= 0, "d3_kv_write: tokens must be >= 0");
  if (tokens == 0) return D3_OK;
  D3_CHECK_ARG(slots, "d3_kv_write: null slots");
  if ((rc = check_rows(k, k_token, k_head, "d3_kv_write: k"))) return rc;
  if ((rc = check_rows(v, v_token, v_head, "d3_kv_write: v"))) return rc;
  FillParams p{};
  p.k = RowsIn{k, k_token, k_head};
  p.v = RowsIn{v, v_token, v_head};
  p.slots = slots;
  p.slot_bytes = slot_bytes;
  p.tokens = tokens;
  p.kv_heads = cache->kv_heads;
  p.cache = *cache;
  p.tokens_per_cta = tokens_per_cta(tokens);
  return dtype == D3_BF16 ? launch_fill<__nv_bfloat16>(p, cache->head_dim, false, (cudaStream_t)stream)
                          : launch_fill<__half>(p, cache->head_dim, false, (cudaStream_t)stream);
}

int d3_kv_read(const d3_kv_cache* cache, const void* slots, int32_t slot_bytes, int32_t tokens,
               int32_t dtype, void* k_out, void* v_out, d3_stream_t stream) {
  int rc = check_kv_cache(cache, "d3_kv_read");
  if (rc) return rc;
  D3_CHECK_ARG(dtype == D3_BF16 || dtype == D3_F16, "d3_kv_read: rows must be bf16 or fp16");
  D3_CHECK_ARG(cache->dtype == D3_E4M3 || cache->dtype == dtype,
               "d3_kv_read: a 16-bit cache gives rows of its own type");
  D3_CHECK_ARG(slot_bytes == 4 || slot_bytes == 8, "slot_bytes must be 4 or 8");
  D3_CHECK_ARG(tokens >= 0, "d3_kv_read: tokens must be >= 0");
  if (tokens == 0) return D3_OK;
  D3_CHECK_ARG(slots && k_out && v_out, "d3_kv_read: null pointer");
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(D3_ERR_MISALIGNED, "d3_kv_read: outputs not 16-byte aligned");
  ReadParams p{slots, slot_bytes, tokens, k_out, v_out, *cache};
  const int D = cache->head_dim;
  const long long rows = 2LL * cache->kv_heads * tokens, per = 256 / (D / 8) * kReadRows;
  if ((rows + per - 1) / per >= (1LL << 31))
    return fail(D3_ERR_TOO_LARGE, "d3_kv_read: too many rows");
  const dim3 grid((unsigned)((rows + per - 1) / per));
  void (*kern)(ReadParams) = dtype == D3_BF16 ? (D == 128 ? kv_read_kernel<__nv_bfloat16, 128> : kv_read_kernel<__nv_bfloat16, 256>)
                                              : (D == 128 ? kv_read_kernel<__half, 128> : kv_read_kernel<__half, 256>);
  D3_CUDA_TRY(launch_k(kern, grid, dim3(256), 0, (cudaStream_t)stream, pdl_enabled(), p),
              "kv_read_kernel launch");
  return D3_OK;
}

int d3_qk_norm_rope(const d3_norm_rope* a, const d3_kv_cache* cache, d3_stream_t stream) {
  D3_CHECK_ARG(a, "d3_qk_norm_rope: null arguments");
  int rc;
  if (cache && (rc = check_kv_cache(cache, "d3_qk_norm_rope"))) return rc;
  D3_CHECK_ARG(a->dtype == D3_BF16 || a->dtype == D3_F16,
               "d3_qk_norm_rope: rows must be bf16 or fp16");
  D3_CHECK_ARG(a->tokens >= 0 && a->heads >= 1 && a->kv_heads >= 1,
               "d3_qk_norm_rope: tokens must be >= 0, heads and kv_heads >= 1");
  if (a->head_dim != 128 && a->head_dim != 256)
    return fail(D3_ERR_UNSUPPORTED, "d3_qk_norm_rope: head_dim %d (128 or 256)", (int)a->head_dim);
  if (a->rotary_dim < 16 || a->rotary_dim > a->head_dim || a->rotary_dim % 16)
    return fail(D3_ERR_UNSUPPORTED, "d3_qk_norm_rope: rotary_dim %d (a multiple of 16 in 16..head_dim)",
                (int)a->rotary_dim);
  D3_CHECK_ARG((a->pos_bytes == 4 || a->pos_bytes == 8), "pos_bytes must be 4 or 8");
  D3_CHECK_ARG(a->eps >= 0.f, "d3_qk_norm_rope: eps must be >= 0");
  if (cache) {
    D3_CHECK_ARG(cache->kv_heads == a->kv_heads && cache->head_dim == a->head_dim,
                 "d3_qk_norm_rope: the cache has other heads");
    D3_CHECK_ARG(cache->dtype == D3_E4M3 || cache->dtype == a->dtype,
                 "d3_qk_norm_rope: a 16-bit cache takes rows of its own type");
    D3_CHECK_ARG(a->slot_bytes == 4 || a->slot_bytes == 8, "slot_bytes must be 4 or 8");
  }
  if (a->tokens == 0) return D3_OK;
  D3_CHECK_ARG(a->positions && a->inv_freq && a->q_weight && a->k_weight && (!cache || a->slots),
               "d3_qk_norm_rope: null pointer");
  if ((rc = check_rows(a->q, a->q_token, a->q_head, "d3_qk_norm_rope: q"))) return rc;
  if ((rc = check_rows(a->k, a->k_token, a->k_head, "d3_qk_norm_rope: k"))) return rc;
  if ((rc = check_rows(a->q_out, a->q_out_token, a->q_out_head, "d3_qk_norm_rope: q_out"))) return rc;
  if (cache && (rc = check_rows(a->v, a->v_token, a->v_head, "d3_qk_norm_rope: v"))) return rc;
  if (!cache && (rc = check_rows(a->k_out, a->k_out_token, a->k_out_head, "d3_qk_norm_rope: k_out")))
    return rc;
  if (!aligned16(a->q_weight) || !aligned16(a->k_weight))
    return fail(D3_ERR_MISALIGNED, "d3_qk_norm_rope: weights not 16-byte aligned");
  FillParams p{};
  p.q = RowsIn{a->q, a->q_token, a->q_head};
  p.k = RowsIn{a->k, a->k_token, a->k_head};
  p.v = RowsIn{a->v, a->v_token, a->v_head};
  p.q_out = a->q_out;
  p.q_out_token = a->q_out_token;
  p.q_out_head = a->q_out_head;
  p.k_out = a->k_out;
  p.k_out_token = a->k_out_token;
  p.k_out_head = a->k_out_head;
  p.q_w = a->q_weight;
  p.k_w = a->k_weight;
  p.positions = a->positions;
  p.pos_bytes = a->pos_bytes;
  p.inv_freq = a->inv_freq;
  p.slots = a->slots;
  p.slot_bytes = a->slot_bytes;
  p.tokens = a->tokens;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.half = a->rotary_dim / 2;
  p.interleaved = a->interleaved;
  p.eps = a->eps;
  p.w_offset = a->weight_offset;
  if (cache) p.cache = *cache;
  else p.cache.dtype = a->dtype;
  p.tokens_per_cta = tokens_per_cta(a->tokens);
  return a->dtype == D3_BF16 ? launch_fill<__nv_bfloat16>(p, a->head_dim, true, (cudaStream_t)stream)
                             : launch_fill<__half>(p, a->head_dim, true, (cudaStream_t)stream);
}

}  // extern "C"
