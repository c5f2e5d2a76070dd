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
  int pos_bytes, slot_bytes, tokens, heads, kv_heads, half, interleaved, page_shift;
  int tokens_per_cta;
  float eps, w_offset;
  d3_kv_cache cache;      // k == NULL: no cache
};

constexpr int kFillThreads = 256;
constexpr int kMaxHalf = 128;          // rotary pairs of the widest head
constexpr int kMaxTokensPerCta = 8;

// x / s rounded as the division is.  With r = 1 / s rounded and q = x r, the
// remainder q s - x is exact in one fused step and q - rem r is the quotient
// rounded correctly (Markstein's correction): three operations, two values at
// a time, where a division takes about ten.  The remainder must not
// underflow: the caller sees to it that s is not far from 1.  (With the
// remainder's sign the other way round -0 would become 0.)
__device__ __forceinline__ void div2(float& x, float& y, float s, float r) {
  float q0 = x, q1 = y;
  mul2(q0, q1, r, r);
  x = -x;
  y = -y;
  fma2v(x, y, q0, s, q1, s);
  fma2v(q0, q1, x, -r, y, -r);
  x = q0;
  y = q1;
}

// Where a group of lanes is among rows of `per` a token: token t, row h.
struct At {
  int t, h;
  __device__ __forceinline__ void advance(int by, int per) {
    h += by;
    while (h >= per) {
      h -= per;
      ++t;
    }
  }
};

// One cached row: 8 elements a lane of D / 8.
template <typename T, int D, bool E4>
__device__ __forceinline__ void put_row(void* buf, float* scales, long long row, int lane, float (&y)[8], bool live) {
  constexpr int L = D / 8;
  if (E4) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float s;
    uint32_t w[4];
    if (amax > 0x1p-80f && amax < 0x1p120f) {
      s = amax;
      float unused = amax;
      div2(s, unused, kE4m3Max, 1.f / kE4m3Max);
      const float r = __frcp_rn(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        div2(y[2 * i], y[2 * i + 1], s, r);
        w[i] = e4m3x2(y[2 * i], y[2 * i + 1]);
      }
    } else {      // zeros, infinities, the ends of the range
      s = amax > 0.f ? amax / kE4m3Max : 1.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = e4m3x2(y[2 * i] / s, y[2 * i + 1] / s);
    }
    if (live) {
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(buf) + row * D + lane * 8) =
          make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
      if (lane == 0) scales[row] = s;
    }
  } else if (live) {
    *reinterpret_cast<uint4*>(static_cast<T*>(buf) + row * D + lane * 8) = pack8<T>(y);
  }
}

// A group of D/8 lanes holds a row; NORM: norm and rotation of q and k rows
// (otherwise there are no q rows and K goes in as it is).  E4: K and V become
// codes.  Queries first, then K and V of a token and head together, which
// share their place; what a row does not need (a query's largest value, a
// value's norm) is not computed: the kernel is as much bound by its
// instructions as by HBM (8192 tokens of 16 + 2 heads of 256 into codes: 46 us,
// 4.0 TB/s, 75 % of the issue slots).  Five blocks an SM leave 48 registers, of
// which the variants with the norm spill 56 to 68 bytes.
template <typename T, int D, bool NORM, bool E4>
__global__ void __launch_bounds__(kFillThreads, 5) kv_fill_kernel(const __grid_constant__ FillParams p) {
  constexpr int L = D / 8;                          // lanes of a row
  constexpr int GROUPS = kFillThreads / L;
  __shared__ __align__(16) float s_cos[kMaxTokensPerCta][kMaxHalf], s_sin[kMaxTokensPerCta][kMaxHalf];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const int t0 = blockIdx.x * p.tokens_per_cta;
  const int nt = min(p.tokens_per_cta, p.tokens - t0);
  pdl_trigger();
  pdl_wait();
  auto fetch = [&](const RowsIn& in, At at) {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (at.t < nt)
      u = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(in.p) + (long long)(t0 + at.t) * in.token +
                                                at.h * in.head + lane * 8));
    return u;
  };
  const int n16 = p.half / 8;                       // lanes of one half of the rotated dims
  const bool first = lane < n16;
  const float sign = first ? -1.f : 1.f;
  const int j8 = (first ? lane : lane - n16) * 8;
  // all lanes: norm with weights w, rotation by token t
  auto turn = [&](float (&y)[8], const float (&w)[8], int t) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma2v(s0, s1, y[i], y[i], y[i + 1], y[i + 1]);
    float ss = s0 + s1;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      mul2(y[i], y[i + 1], inv, inv);
      mul2(y[i], y[i + 1], w[i], w[i + 1]);
    }
    const float *cs = s_cos[t], *sn = s_sin[t];
    if (p.interleaved) {
      if (lane * 4 < p.half) {
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
      if (lane < 2 * n16) {
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
  };
  float w[8];
  // the lanes of a warp leave a loop together: the shuffles are whole
  if (NORM) {
    At at{0, 0};
    at.advance(grp, p.heads);
    uint4 raw = fetch(p.q, at);
    for (int i = threadIdx.x; i < nt * p.half; i += kFillThreads) {
      const int t = i / p.half, j = i - t * p.half;
      const double turns = (double)load_index(p.positions, p.pos_bytes, t0 + t) * p.inv_freq[j] *
                           0.15915494309189533577;  // 1 / (2 pi)
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      s_cos[t][j] = c;
      s_sin[t][j] = s;
    }
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p.q_w) + lane * 8), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] += p.w_offset;
    __syncthreads();
    while (__any_sync(0xffffffffu, at.t < nt)) {
      float y[8];
      unpack8<T>(raw, y);
      const At now = at;
      at.advance(GROUPS, p.heads);
      raw = fetch(p.q, at);
      const bool live = now.t < nt;
      turn(y, w, live ? now.t : 0);
      if (live)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.q_out) + (long long)(t0 + now.t) * p.q_out_token +
                                  now.h * p.q_out_head + lane * 8) = pack8<T>(y);
    }
    unpack8<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p.k_w) + lane * 8), w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] += p.w_offset;
  }
  const bool cached = p.cache.k != nullptr;
  const long long slots = (long long)p.cache.pages << p.page_shift;
  At at{0, 0};
  at.advance(grp, p.kv_heads);
  auto fetch_slot = [&](At a) {
    return cached && a.t < nt ? load_index(p.slots, p.slot_bytes, t0 + a.t) : -1;
  };
  uint4 raw_k = fetch(p.k, at), raw_v = make_uint4(0, 0, 0, 0);
  if (cached) raw_v = fetch(p.v, at);
  long long next_slot = fetch_slot(at);
  while (__any_sync(0xffffffffu, at.t < nt)) {
    float k[8], v[8];
    unpack8<T>(raw_k, k);
    unpack8<T>(raw_v, v);
    const At now = at;
    const long long slot = next_slot;
    at.advance(GROUPS, p.kv_heads);
    raw_k = fetch(p.k, at);
    if (cached) raw_v = fetch(p.v, at);
    next_slot = fetch_slot(at);
    if (NORM) turn(k, w, now.t < nt ? now.t : 0);
    if (!cached) {
      if (now.t < nt)
        *reinterpret_cast<uint4*>(static_cast<T*>(p.k_out) + (long long)(t0 + now.t) * p.k_out_token +
                                  now.h * p.k_out_head + lane * 8) = pack8<T>(k);
      continue;
    }
    const bool live = slot >= 0 && slot < slots;
    const long long row = (((slot >> p.page_shift) * p.cache.kv_heads + now.h) << p.page_shift) + (slot & (p.cache.page_size - 1));
    put_row<T, D, E4>(p.cache.k, p.cache.k_scale, row, lane, k, live);
    put_row<T, D, E4>(p.cache.v, p.cache.v_scale, row, lane, v, live);
  }
}

struct ReadParams {
  const void* slots;
  int slot_bytes, tokens, page_shift;
  void *k_out, *v_out;    // [tokens][kv_heads][D], contiguous
  d3_kv_cache cache;
};

constexpr int kReadRows = 2;   // rows a lane group has in flight

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
    const int page = (int)slot[i] >> p.page_shift, off = (int)slot[i] & (p.cache.page_size - 1);
    const long long row = (((long long)page * p.cache.kv_heads + (h2[i] >> 1)) << p.page_shift) + off;
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

// Tokens a CTA takes: one for small batches, which so spread over the SMs;
// four, then eight, once every SM still has several CTAs (8192 tokens of 20
// rows of 256: 53 us with two, 46 with four; 50001 of 16 rows of 128: 64 us
// with four, 60 with eight).
static int tokens_per_cta(int tokens) {
  const int n = num_sms();
  return tokens >= 64 * n ? 8 : tokens >= 8 * n ? 4 : 1;
}

template <typename T, int D>
static void (*fill_kernel(bool norm, bool e4))(FillParams) {
  return norm ? (e4 ? kv_fill_kernel<T, D, true, true> : kv_fill_kernel<T, D, true, false>)
              : (e4 ? kv_fill_kernel<T, D, false, true> : kv_fill_kernel<T, D, false, false>);
}

template <typename T>
static int launch_fill(FillParams p, int D, bool norm, cudaStream_t st) {
  if (p.cache.k) p.page_shift = __builtin_ctz((unsigned)p.cache.page_size);
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
  ReadParams p{slots, slot_bytes, tokens, __builtin_ctz((unsigned)cache->page_size), k_out, v_out, *cache};
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
