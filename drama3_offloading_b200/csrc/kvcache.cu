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

// x / s of a row, rounded as the division is.  With r = 1 / s rounded and
// q = x r, the remainder x - q s is exact in one fused step and q + rem r is
// the quotient rounded correctly (Markstein's correction): three operations
// where a division takes about ten.  The remainder must not underflow, so
// scales far from 1 -- and infinite ones -- take the division.
struct RowDiv {
  float s, r;
  bool plain;
  __device__ __forceinline__ explicit RowDiv(float scale) : s(scale), r(1.f / scale) {
    plain = !(scale > 0x1p-90f && scale < 0x1p119f);
  }
  __device__ __forceinline__ void two(float& x, float& y) const {
    float q0 = x, q1 = y, e0 = x, e1 = y;
    mul2(q0, q1, r, r);
    fma2v(e0, e1, -q0, s, -q1, s);
    fma2v(q0, q1, e0, r, e1, r);
    x = q0;
    y = q1;
  }
};

// A group of D/8 lanes holds one row, ROWS rows at a time, the next ROWS on
// their way; NORM: norm and rotation of q and k rows (otherwise there are no q
// rows and K goes in as it is).  E4: K and V become codes.  What a row does
// not need (a query's largest value, a value's norm) its warp skips: the
// kernel is as much bound by its instructions as by HBM.
template <typename T, int D, bool NORM, bool E4>
__global__ void __launch_bounds__(kFillThreads) kv_fill_kernel(const __grid_constant__ FillParams p) {
  constexpr int L = D / 8;                          // lanes of a row
  constexpr int ROWS = 2;
  constexpr int GROUPS = kFillThreads / L;
  __shared__ __align__(16) float s_cos[kMaxTokensPerCta][kMaxHalf], s_sin[kMaxTokensPerCta][kMaxHalf];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const int t0 = blockIdx.x * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.tokens - t0);
  pdl_trigger();
  float wq[8], wk[8];
  if (NORM) {       // weights are no earlier launch's work
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p.q_w) + lane * 8), wq);
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p.k_w) + lane * 8), wk);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wq[i] += p.w_offset;
      wk[i] += p.w_offset;
    }
  }
  pdl_wait();
  const bool cached = p.cache.k != nullptr;
  const int rows = p.heads + (cached ? 2 : 1) * p.kv_heads;   // q, k and, into a cache, v
  // a group's rows, in order: token t, row h of the token
  struct At {
    int t, h;
  };
  auto next = [&](At a) {
    a.h += GROUPS;
    while (a.h >= rows) {
      a.h -= rows;
      ++a.t;
    }
    return a;
  };
  At ahead{0, grp - GROUPS};
  ahead = next(ahead);
  uint4 raw[ROWS];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      raw[u] = make_uint4(0, 0, 0, 0);
      if (ahead.t < nt) {
        const int k0 = ahead.h - p.heads, v0 = k0 - p.kv_heads;
        const RowsIn& in = k0 < 0 ? p.q : v0 < 0 ? p.k : p.v;
        raw[u] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(in.p) + (long long)(t0 + ahead.t) * in.token +
                                                       (k0 < 0 ? ahead.h : v0 < 0 ? k0 : v0) * in.head + lane * 8));
      }
      ahead = next(ahead);
    }
  };
  At at = ahead;
  load();
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
  const int n16 = p.half / 8;                       // lanes of one half of the rotated dims
  const bool first = lane < n16;
  const float sign = first ? -1.f : 1.f;
  const int j8 = (first ? lane : lane - n16) * 8;
  const long long slots = (long long)p.cache.pages * p.cache.page_size;
  // the lanes of a warp leave together: the shuffles are whole
  while (__any_sync(0xffffffffu, at.t < nt)) {
    float x[ROWS][8];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) unpack8<T>(raw[u], x[u]);
    load();
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const bool live = at.t < nt;
      const int t = live ? at.t : 0, h = at.h, k0 = h - p.heads, v0 = k0 - p.kv_heads;
      const bool is_q = k0 < 0, is_v = v0 >= 0;
      at = next(at);
      const long long tok = t0 + t;
      long long slot = -1;
      if (live && cached && !is_q) slot = load_index(p.slots, p.slot_bytes, tok);
      float (&y)[8] = x[u];
      if (NORM && __any_sync(0xffffffffu, !is_v)) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) fma2v(s0, s1, y[i], y[i], y[i + 1], y[i + 1]);
        float ss = s0 + s1;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!is_v) {
          const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            mul2(y[i], y[i + 1], inv, inv);
            mul2(y[i], y[i + 1], is_q ? wq[i] : wk[i], is_q ? wq[i + 1] : wk[i + 1]);
          }
        }
        const float *cs = s_cos[t], *sn = s_sin[t];
        if (p.interleaved) {
          if (!is_v && lane * 4 < p.half) {
            const float4 c4 = *reinterpret_cast<const float4*>(cs + lane * 4);
            const float4 s4 = *reinterpret_cast<const float4*>(sn + lane * 4);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float a = y[2 * i], b = y[2 * i + 1];
              y[2 * i] = a * c[i] - b * s[i];
              y[2 * i + 1] = b * c[i] + a * s[i];
            }
          }
        } else {
          // lanes [0, R/16) hold the first halves, the next R/16 the second
          float z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            z[i] = __shfl_sync(0xffffffffu, y[i], first ? lane + n16 : lane - n16, L);
          if (!is_v && lane < 2 * n16) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 c = *reinterpret_cast<const float4*>(cs + j8 + i);
              const float4 s = *reinterpret_cast<const float4*>(sn + j8 + i);
              mul2(y[i], y[i + 1], c.x, c.y);
              mul2(y[i + 2], y[i + 3], c.z, c.w);
              mul2(z[i], z[i + 1], sign, sign);
              mul2(z[i + 2], z[i + 3], sign, sign);
              fma2v(y[i], y[i + 1], z[i], s.x, z[i + 1], s.y);
              fma2v(y[i + 2], y[i + 3], z[i + 2], s.z, z[i + 3], s.w);
            }
          }
        }
      }
      float amax = 0.f;
      if (E4 && __any_sync(0xffffffffu, !is_q)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1)
          amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      }
      if (!live) continue;
      if (is_q) {
        *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + tok * p.q_out_token +
                                  h * p.q_out_head + lane * 8) = pack8<T>(y);
        continue;
      }
      if (!cached) {
        *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + tok * p.k_out_token +
                                  k0 * p.k_out_head + lane * 8) = pack8<T>(y);
        continue;
      }
      if (slot < 0 || slot >= slots) continue;
      const int page = (int)slot / p.cache.page_size, off = (int)slot - page * p.cache.page_size;
      const long long row = ((long long)page * p.cache.kv_heads + (is_v ? v0 : k0)) * p.cache.page_size + off;
      void* base = is_v ? p.cache.v : p.cache.k;
      if (E4) {
        const float s = amax > 0.f ? amax / kE4m3Max : 1.f;
        const RowDiv div(s);
        uint32_t w[4];
        if (div.plain) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = e4m3x2(y[2 * i] / s, y[2 * i + 1] / s);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            div.two(y[2 * i], y[2 * i + 1]);
            w[i] = e4m3x2(y[2 * i], y[2 * i + 1]);
          }
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(base) + row * D + lane * 8) =
            make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
        if (lane == 0) (is_v ? p.cache.v_scale : p.cache.k_scale)[row] = s;
      } else {
        *reinterpret_cast<uint4*>(static_cast<T*>(base) + row * D + lane * 8) = pack8<T>(y);
      }
    }
  }
}

struct ReadParams {
  const void* slots;
  int slot_bytes, tokens;
  void *k_out, *v_out;    // [tokens][kv_heads][D], contiguous
  d3_kv_cache cache;
};

constexpr int kReadRows = 4;   // rows a lane group has in flight

// Rows of the cache back in 16 bits: T(code * s), or the row as it is.  A lane
// takes 16 bytes of a row.
template <typename T, int D, bool E4>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int PER = E4 ? 16 : 8, L = D / PER, GROUPS = 256 / L;
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  pdl_trigger();
  pdl_wait();
  const int per = 2 * p.cache.kv_heads;
  const long long rows = (long long)p.tokens * per;
  const long long r0 = (long long)blockIdx.x * (GROUPS * kReadRows) + grp;
  bool live[kReadRows], have[kReadRows];
  uint4 raw[kReadRows];
  float sc[kReadRows];
  long long to[kReadRows], slot[kReadRows];
  int h2[kReadRows];
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const long long r = r0 + i * GROUPS;
    live[i] = r < rows;
    const int t = live[i] ? (int)((unsigned)r / (unsigned)per) : 0;
    h2[i] = (int)r - t * per;
    to[i] = ((long long)t * p.cache.kv_heads + (h2[i] >> 1)) * D + lane * PER;
    slot[i] = live[i] ? load_index(p.slots, p.slot_bytes, t) : -1;
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    have[i] = slot[i] >= 0 && slot[i] < (long long)p.cache.pages * p.cache.page_size;
    raw[i] = make_uint4(0, 0, 0, 0);
    sc[i] = 0.f;
    if (!have[i]) continue;
    const int page = (int)slot[i] / p.cache.page_size, off = (int)slot[i] - page * p.cache.page_size;
    const long long row = ((long long)page * p.cache.kv_heads + (h2[i] >> 1)) * p.cache.page_size + off;
    const bool v = h2[i] & 1;
    raw[i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(v ? p.cache.v : p.cache.k) +
                                                   row * (D * (E4 ? 1 : 2)) + lane * 16));
    if (E4) sc[i] = __ldcg((v ? p.cache.v_scale : p.cache.k_scale) + row);
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    if (!live[i]) continue;
    T* out = static_cast<T*>(h2[i] & 1 ? p.v_out : p.k_out) + to[i];
    if (E4) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = e4m3x2_to_f2((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
        o[j] = have[i] ? Elem<T>::from_f2(f.x * sc[i], f.y * sc[i]) : 0u;
      }
      *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4*>(out + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      *reinterpret_cast<uint4*>(out) = raw[i];
    }
  }
}

// ---------------------------------------------------------------- host

// Tokens a CTA takes: one for small batches (as many CTAs as tokens, so that
// a decode batch spreads over the SMs), four once there are enough tokens for
// every SM to hold several CTAs all the same.
static int tokens_per_cta(int tokens) { return tokens >= 8 * num_sms() ? kMaxTokensPerCta : 1; }

template <typename T, int D>
static void (*fill_kernel(bool norm, bool e4))(FillParams) {
  return norm ? (e4 ? kv_fill_kernel<T, D, true, true> : kv_fill_kernel<T, D, true, false>)
              : (e4 ? kv_fill_kernel<T, D, false, true> : kv_fill_kernel<T, D, false, false>);
}

template <typename T>
static int launch_fill(const FillParams& p, int D, bool norm, cudaStream_t st) {
  const dim3 grid((unsigned)((p.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta));
  const bool e4 = p.cache.dtype == D3_E4M3;
  void (*k)(FillParams) = D == 128 ? fill_kernel<T, 128>(norm, e4) : fill_kernel<T, 256>(norm, e4);
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
  const int D = cache->head_dim, lanes = D / (cache->dtype == D3_E4M3 ? 16 : 8);
  const long long rows = 2LL * cache->kv_heads * tokens, per = 256 / lanes * kReadRows;
  if (rows >= (1LL << 31)) return fail(D3_ERR_TOO_LARGE, "d3_kv_read: too many rows");
  const dim3 grid((unsigned)((rows + per - 1) / per));
  const bool e4 = cache->dtype == D3_E4M3;
  void (*kern)(ReadParams) =
      dtype == D3_BF16 ? (D == 128 ? (e4 ? kv_read_kernel<__nv_bfloat16, 128, true> : kv_read_kernel<__nv_bfloat16, 128, false>)
                                   : (e4 ? kv_read_kernel<__nv_bfloat16, 256, true> : kv_read_kernel<__nv_bfloat16, 256, false>))
                       : (D == 128 ? (e4 ? kv_read_kernel<__half, 128, true> : kv_read_kernel<__half, 128, false>)
                                   : (e4 ? kv_read_kernel<__half, 256, true> : kv_read_kernel<__half, 256, false>));
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
