// Attention of a chunk of new tokens over a paged K/V cache, on the tensor
// cores: a CTA pair (tcgen05, cta_group::2) holds 256 query rows of one KV
// head -- 2 * (128 / G) tokens times the G query heads that share it -- and
// walks the keys in blocks of 128 with a running maximum and sum:
//
//   S [256 x 128] = Q K^T       (both operands in shared memory)
//   P = exp2(S * c - m)         (each thread one row, TMEM -> TMEM)
//   O [256 x D] += P V          (P from TMEM, V from shared memory)
//
// Why a pair: per 128-key block a CTA's tensor core needs 8 D cycles for 128
// rows, and K and V of the block are 512 D bytes -- 64 bytes a cycle for every
// SM, which L2 does not deliver to all of them at once.  In a pair each CTA
// loads half of K (64 keys) and half of V (D/2 dims) and the pair's MMAs read
// both halves: 32 bytes a cycle, and twice as many blocks fit in the ring.
//
// Bound: the tensor pipe for D = 256 (2048 cycles a block against about 1300
// for the exponentials of 128 x 128 scores on one warpgroup); the
// exponentials for D = 128.
//
// TMEM, 512 columns: two S blocks (P overwrites its own S) and O.  S of block
// j + 1 is issued before P V of block j, so the tensor core works while the
// softmax does.  O is only rescaled when a row's maximum grows by more than 8
// (in log2): P then stays below 2^8, sums are in fp32 and the quotient of the
// two does not change.
//
// Roles (per CTA): warps 0-3 softmax and output, warp 4 issues the MMAs (in
// the pair's first CTA), warp 5 the TMA loads; for codes warps 6-9 load,
// widen and store the tiles themselves.
//
// A block's last page, when the sequence ends in it, is loaded shifted: rows
// before the page's first come from outside the tensor map and are zeros, the
// page's valid rows follow, and what lies behind the end (NaN, perhaps) never
// reaches shared memory.  The mask knows about the shift.
//
// Split: as in the row kernel, the list of all (sequence, KV head, row tile,
// key block) is cut into equal parts, one per pair; tiles that a cut goes
// through are joined by attn_chunk_join_kernel in the parts' order.
//
// e4m3 caches: K codes are exact in 16 bits and their scale multiplies a
// column of S in fp32; V is widened to T(code * scale), as kvcache.read gives
// it.
#pragma once

#include "attn_rows.cuh"

namespace d3 {

constexpr int kAttnErrChunkLoad = 53, kAttnErrChunkMma = 54, kAttnErrChunkSoftmax = 55,
              kAttnErrChunkWiden = 56;
constexpr int kBlockKeys = 128;
constexpr float kRescaleLog2 = 8.f;

template <typename T, int D, bool E4>
struct ChunkCfg {
  static constexpr int THREADS = E4 ? 320 : 192;
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int SLOT = 64 * D * 2;                 // half a block of K or of V
  static constexpr int SLOTS = E4 ? (D == 256 ? 4 : 8) : (D == 256 ? 5 : 10);
  static constexpr int KS_RING = 8;                       // K scales of 8 blocks
  static constexpr int KS_BYTES = E4 ? KS_RING * kBlockKeys * 4 : 0;
  static constexpr size_t SMEM = 1024 + Q_BYTES + (size_t)SLOTS * SLOT + KS_BYTES + 512;
  static constexpr int COL_S = 0, COL_O = 256;
  // K scales of block j + KS_RING are written no earlier than the slot of V of
  // block j is free, when its softmax is over
  static_assert(2 * KS_RING >= SLOTS + 3, "K scale ring too short");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct ChunkWs {           // carved from the call's workspace
  float* o;                // [pairs][2][256][D]
  float* ml;               // [pairs][2][256][2]
  int4* desc;              // [pairs]: sequence, KV head, row tile, last part (-1: none)
};

// sum of floor((a i + b) / m) over i in [0, n), all arguments >= 0: the
// Euclid-like reduction of a lattice point count
__device__ __forceinline__ long long floor_sum(long long n, long long m, long long a, long long b) {
  long long ans = 0;
  if (n <= 0) return 0;
  while (true) {
    if (a >= m) {
      ans += (n - 1) * n / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      ans += n * (b / m);
      b %= m;
    }
    const long long y = a * n + b;
    if (y < m) return ans;
    n = y / m;
    b = y % m;
    const long long t = m;
    m = a;
    a = t;
  }
}

// key blocks that row tile i (of `per` tokens) of a sequence sees: at least one
__device__ __forceinline__ int chunk_blocks(const AttnSeq& s, int per, int i) {
  const int vis = s.kv - s.n + min((i + 1) * per, s.n);
  return max(1, (vis + kBlockKeys - 1) / kBlockKeys);
}
// ... of row tiles [0, i), i below the sequence's number of tiles
__device__ __forceinline__ long long chunk_before(const AttnSeq& s, int per, int i) {
  const long long base = s.kv - s.n;
  long long ones = base >= kBlockKeys ? 0 : (kBlockKeys - base) / per;
  ones = ones < i ? ones : i;
  return ones + floor_sum(i - ones, kBlockKeys, per, base + (ones + 1) * per + kBlockKeys - 1);
}
__device__ __forceinline__ int chunk_tiles(const AttnSeq& s, int per) { return (s.n + per - 1) / per; }
__device__ __forceinline__ long long chunk_head_units(const AttnSeq& s, int per) {
  const int nq = chunk_tiles(s, per);
  return chunk_before(s, per, nq - 1) + chunk_blocks(s, per, nq - 1);
}
__device__ __forceinline__ bool chunk_takes(const AttnParams& p, const AttnSeq& s) {
  return s.rows > 0 && s.rows >= p.min_rows && s.rows <= p.max_rows;
}

struct ChunkPiece {
  AttnSeq s;
  int b, head, tile, j0, j1, nb;
};
struct ChunkWalk {
  int b;
  long long left, off;
  bool fresh;             // at the start of a part: (head, tile) not known yet
  int head, tile, j;
  AttnSeq s;
  __device__ __forceinline__ bool next(const AttnParams& p, int per, ChunkPiece& w) {
    if (left <= 0) return false;
    if (fresh) {
      fresh = false;
      s = attn_seq(p, b);
      const long long u = chunk_head_units(s, per);
      head = (int)(off / u);
      const long long r = off - head * u;
      int lo = 0, hi = chunk_tiles(s, per) - 1;      // the last tile that starts at or before r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (chunk_before(s, per, mid) <= r) lo = mid;
        else hi = mid - 1;
      }
      tile = lo;
      j = (int)(r - chunk_before(s, per, lo));
    } else {
      j = 0;
      if (++tile >= chunk_tiles(s, per)) {
        tile = 0;
        if (++head >= p.kv_heads) {
          head = 0;
          do {
            if (++b >= p.batch) return false;
            s = attn_seq(p, b);
          } while (!chunk_takes(p, s));
        }
      }
    }
    w.s = s;
    w.b = b;
    w.head = head;
    w.tile = tile;
    w.nb = chunk_blocks(s, per, tile);
    w.j0 = j;
    w.j1 = (int)min((long long)w.nb, j + left);
    left -= w.j1 - w.j0;
    return true;
  }
};

// ---------------------------------------------------------------- PTX

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same shared-memory address in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if (globaltimer_ns() - t0 > kAttnWaitBudgetNs) return false;
  }
}
// loads of a pair's CTA that complete on a barrier of either CTA; no multicast
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x),
      "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void mma_pair_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_pair_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// arrives on the barrier at this address in both CTAs once all MMAs issued so far are done
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t a, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of an operand whose contiguous dim is the MMA's N (V: dims), with
// the 128-byte swizzle: 64-element columns `col_bytes` apart, groups of eight
// k rows 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_n128(uint32_t saddr, uint32_t col_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((col_bytes >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
// kind::f16, D in fp32, A and B both bf16 or both fp16
template <typename T>
__device__ constexpr uint32_t idesc_16(int M, int N, bool b_n_major) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// two codes as two T values
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint16_t c);
template <>
__device__ __forceinline__ uint32_t widen2<__half>(uint16_t c) { return e4m3x2_to_h2(c); }
template <>
__device__ __forceinline__ uint32_t widen2<__nv_bfloat16>(uint16_t c) {
  const float2 f = e4m3x2_to_f2(c);
  return Elem<__nv_bfloat16>::from_f2(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint16_t c, float s) {
  const float2 f = e4m3x2_to_f2(c);
  return Elem<T>::from_f2(f.x * s, f.y * s);
}

// ---------------------------------------------------------------- kernel

template <typename T, int D, bool E4>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ChunkCfg<T, D, E4>::THREADS, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p,
                      const ChunkWs ws) {
  using C = ChunkCfg<T, D, E4>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_scan[33];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sq = smem_u32(smem), ss = sq + C::Q_BYTES;
  float* s_ks = reinterpret_cast<float*>(smem + C::Q_BYTES + (size_t)C::SLOTS * C::SLOT);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::Q_BYTES + (size_t)C::SLOTS * C::SLOT + C::KS_BYTES);
  uint64_t* empty = full + C::SLOTS;
  uint64_t* q_full = empty + C::SLOTS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;        // [2]
  uint64_t* p_ready = s_full + 2;        // [2]
  uint64_t* o_done = p_ready + 2;
  uint64_t* o_free = o_done + 1;
  uint64_t* o_last = o_free + 1;
  uint64_t* all_done = o_last + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, E4 ? 8 : 1);   // E4: four warps of either CTA
      mbar_init(empty + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 8);         // four warps of either CTA
    }
    mbar_init(o_done, 1);
    mbar_init(o_free, 8);
    mbar_init(o_last, 1);
    mbar_init(all_done, 1);
    fence_barrier_init();
    s_abort = 0;
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_trigger();
  pdl_wait();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tpc = 128 / p.group, per = 2 * tpc;      // tokens of a CTA, of the pair
  const RowsWork work = list_plan(
      p, s_scan,
      [&](int b) -> long long {
        const AttnSeq s = attn_seq(p, b);
        return chunk_takes(p, s) ? chunk_head_units(s, per) * p.kv_heads : 0;
      },
      [&](RowsWork& r) {
        const long long g = min((long long)pairs, r.total);
        r.begin = pair < g ? r.total * pair / g : 0;
        r.count = pair < g ? r.total * (pair + 1) / g - r.begin : 0;
      });
  cluster_sync_all();      // both CTAs' barriers are ready
  ChunkWalk walk;
  walk.b = work.b;
  walk.left = work.count;
  walk.off = work.off;
  walk.fresh = true;
  ChunkPiece w;
  const int ps = p.page_size;

  if (warp == 5 && !E4) {
    // ---- TMA: Q of a piece, then K0, K1, V0, K2, V1, ..., V last
    int slot = 0;
    uint32_t phase = 0, qn = 0;
    bool ok = true;
    const int kbox = min(ps, 64), vbox = min(ps, kBlockKeys);
    auto load = [&](const ChunkPiece& x, int j, bool is_v) {
      if (ok && !mbar_wait(empty + slot, phase ^ 1, kAttnWaitBudgetNs)) {
        if (lane == 0) attn_error(p.err, kAttnErrChunkLoad);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok && !s_abort);
      if (!ok) return;
      if (rank == 0 && lane == 0) mbar_arrive_expect_tx(full + slot, 2 * C::SLOT);
      __syncwarp();
      const uint32_t bar = mapa(smem_u32(full + slot), 0);
      const uint32_t dst = ss + slot * C::SLOT;
      // boxes of one column, columns of 64 dims
      const int box = is_v ? vbox : kbox, rows = is_v ? kBlockKeys : 64, n = rows / box;
      const int cols = is_v ? D / 128 : D / 64;
      for (int i = lane; i < n * cols; i += 32) {
        const int bx = i % n, col = i / n;
        const int key = j * kBlockKeys + (is_v ? 0 : 64 * (int)rank) + bx * box;
        const int pg = key >> p.page_shift, start = pg << p.page_shift;
        int z = -1, y = key - start;
        if (start < x.s.kv) {
          const int id = __ldcg(p.table + (long long)x.b * p.table_stride + pg);
          if (id >= 0 && id < p.pages) z = id * p.kv_heads + x.head;
          if (start + ps > x.s.kv) y -= start + ps - x.s.kv;    // the last page: shifted
        }
        // outside the map (no page, or before its first row): zeros
        tma_pair_3d(dst + col * (rows * 128) + bx * (box * 128), is_v ? &tm_v : &tm_k, bar,
                    (is_v ? (int)rank * (D / 2) : 0) + col * 64, y, z);
      }
      if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
    };
    while (ok && walk.next(p, per, w)) {
      if (!mbar_wait(q_empty, (qn & 1) ^ 1, kAttnWaitBudgetNs)) {
        if (lane == 0) attn_error(p.err, kAttnErrChunkLoad);
        ok = false;
      }
      ++qn;
      ok = __all_sync(0xffffffffu, ok && !s_abort);
      if (!ok) break;
      if (lane == 0) {
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * (D / 64) * tpc * p.group * 128);
        const uint32_t bar = mapa(smem_u32(q_full), 0);
        const int tok = w.s.q0 + w.tile * per + (int)rank * tpc;
        for (int c = 0; c < D / 64; ++c)
          tma_pair_3d(sq + c * (128 * 128), &tm_q, bar, c * 64, w.head * p.group, tok);
      }
      __syncwarp();
      for (int j = w.j0; j < w.j1; ++j) {
        load(w, j, false);
        if (j > w.j0) load(w, j - 1, true);
      }
      load(w, w.j1 - 1, true);
    }
    if (!ok) s_abort = 1;
    if (!ok && rank == 0)
      for (int i = 0; i < C::SLOTS; ++i) mbar_wait(full + i, phase ^ (i < slot ? 0 : 1), kAttnWaitBudgetNs);
  } else if (warp == 5) {
    // ---- codes: only Q comes by TMA
    uint32_t qn = 0;
    bool ok = true;
    while (ok && walk.next(p, per, w)) {
      if (!mbar_wait(q_empty, (qn & 1) ^ 1, kAttnWaitBudgetNs)) {
        if (lane == 0) attn_error(p.err, kAttnErrChunkLoad);
        ok = false;
      }
      ++qn;
      ok = __all_sync(0xffffffffu, ok && !s_abort);
      if (!ok) break;
      if (lane == 0) {
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * (D / 64) * tpc * p.group * 128);
        const uint32_t bar = mapa(smem_u32(q_full), 0);
        const int tok = w.s.q0 + w.tile * per + (int)rank * tpc;
        for (int c = 0; c < D / 64; ++c)
          tma_pair_3d(sq + c * (128 * 128), &tm_q, bar, c * 64, w.head * p.group, tok);
      }
      __syncwarp();
    }
    if (!ok) s_abort = 1;
  } else if (warp == 4) {
    // ---- MMAs of the pair
    if (rank == 0 && lane == 0) {
      constexpr uint32_t id_s = idesc_16<T>(256, kBlockKeys, false), id_o = idesc_16<T>(256, D, true);
      int slot = 0;
      uint32_t phase = 0, it = 0, qn = 0, pieces = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t par) {
        if (ok && !mbar_wait_cluster(bar, par)) {
          attn_error(p.err, kAttnErrChunkMma);
          s_abort = 1;
          ok = false;
        }
        ok = ok && !s_abort;
        return ok;
      };
      auto advance = [&]() {
        commit_pair(empty + slot);
        if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
      };
      auto scores = [&](uint32_t x) {
        if (!wait(full + slot, phase)) return;
        tc_fence_after();
        const uint32_t kb = ss + slot * C::SLOT, d = tmem + C::COL_S + (x & 1) * kBlockKeys;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_pair_ss(d, smem_desc_k128(sq + (k >> 2) * (128 * 128) + (k & 3) * 32),
                      smem_desc_k128(kb + (k >> 2) * (64 * 128) + (k & 3) * 32), id_s, k > 0);
        advance();
        commit_pair(s_full + (x & 1));
      };
      auto values = [&](uint32_t x, bool first) {
        if (!wait(p_ready + (x & 1), (x >> 1) & 1)) return;
        if (!wait(full + slot, phase)) return;
        if (first && pieces > 0 && !wait(o_free, (pieces - 1) & 1)) return;
        tc_fence_after();
        const uint32_t vb = ss + slot * C::SLOT, a = tmem + C::COL_S + (x & 1) * kBlockKeys;
#pragma unroll
        for (int k = 0; k < kBlockKeys / 16; ++k)
          mma_pair_ts(tmem + C::COL_O, a + k * 8, smem_desc_n128(vb + k * (16 * 128), kBlockKeys * 128), id_o,
                      !first || k > 0);
        advance();
        commit_pair(o_done);
      };
      while (ok && walk.next(p, per, w)) {
        if (!wait(q_full, qn & 1)) break;
        ++qn;
        for (int j = w.j0; j < w.j1 && ok; ++j, ++it) {
          scores(it);
          if (j == w.j1 - 1 && ok) commit_pair(q_empty);
          if (j > w.j0 && ok) values(it - 1, j - 1 == w.j0);
        }
        if (ok) values(it - 1, w.j1 - 1 == w.j0);
        if (ok) commit_pair(o_last);
        ++pieces;
      }
      commit_pair(all_done);
    }
  } else if (warp < 4) {
    // ---- softmax: thread = row
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const int rr = warp * 32 + lane, ti = rr / p.group;
    const int hd = rr - ti * p.group;
    uint32_t it = 0, pieces = 0;
    bool ok = true;
    int4 desc = make_int4(0, 0, 0, -1);
    const float c = p.scale_log2;
    auto wait = [&](uint64_t* bar, uint32_t par) {
      if (ok && !mbar_wait_cluster(bar, par)) {
        attn_error(p.err, kAttnErrChunkSoftmax);
        s_abort = 1;
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok && !s_abort);
    };
    while (ok && walk.next(p, per, w)) {
      const int tok = w.tile * per + (int)rank * tpc + ti;       // of the sequence's new ones
      const bool row_ok = ti < tpc && tok < w.s.n;
      const int last = row_ok ? w.s.kv - w.s.n + tok : -1;
      float m = -INFINITY, l = 0.f;
      for (int j = w.j0; j < w.j1; ++j, ++it) {
        const uint32_t sb = lanes + C::COL_S + (it & 1) * kBlockKeys;
        wait(s_full + (it & 1), (it >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        float s[kBlockKeys];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(sb + 32 * i, s + 32 * i);
        tmem_ld_wait();
        if (E4) {
          const float4* ks = reinterpret_cast<const float4*>(s_ks + (it % C::KS_RING) * kBlockKeys);
#pragma unroll
          for (int i = 0; i < kBlockKeys / 4; ++i) {
            const float4 f = ks[i];
            s[4 * i] *= f.x;
            s[4 * i + 1] *= f.y;
            s[4 * i + 2] *= f.z;
            s[4 * i + 3] *= f.w;
          }
        }
        const int lim = last - j * kBlockKeys;                    // last visible key of the block
        if (__any_sync(0xffffffffu, lim < kBlockKeys - 1)) {
          // columns from t0 hold the sequence's last page, `shift` columns late
          const int valid = w.s.kv - j * kBlockKeys;
          int t0 = kBlockKeys, shift = 0;
          if (!E4 && valid > 0 && valid < kBlockKeys) {
            t0 = (valid - 1) / ps * ps;
            shift = t0 + ps - valid;
          }
#pragma unroll
          for (int i = 0; i < kBlockKeys; ++i) {
            const int key = i < t0 ? i : (i < t0 + shift ? kBlockKeys : i - shift);
            if (key > lim) s[i] = -INFINITY;
          }
        }
        float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < kBlockKeys; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i]);
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
        const bool grow = mx > m + kRescaleLog2 || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2(m - mx);
          if (grow) m = mx;
          l *= f;
          if (j > w.j0) {
            // one phase to wait for: P V of the block before came before this
            // S, and this block's waits for this warp
            wait(o_done, (it - 1) & 1);
            if (!ok) break;
            tc_fence_after();
            // 32 columns at a time; a row that starts here holds zeros or what
            // its factor 0 must not turn into NaN
#pragma unroll 1
            for (int i = 0; i < D / 32; ++i) {
              float o[32];
              tmem_ld32(lanes + C::COL_O + 32 * i, o);
              tmem_ld_wait();
#pragma unroll
              for (int q = 0; q < 32; ++q) o[q] = f == 0.f ? 0.f : o[q] * f;
              uint32_t u[32];
#pragma unroll
              for (int q = 0; q < 32; ++q) u[q] = __float_as_uint(o[q]);
              tmem_st32(lanes + C::COL_O + 32 * i, u);
            }
            tmem_st_wait();
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        float l2[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t pk[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) {
            const float a = ex2(fmaf(s[64 * i + 2 * q], c, -base)), b = ex2(fmaf(s[64 * i + 2 * q + 1], c, -base));
            l2[0] += a;
            l2[1] += b;
            pk[q] = Elem<T>::from_f2(a, b);
          }
          tmem_st32(sb + 32 * i, pk);
        }
        l += l2[0] + l2[1];
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(p_ready + (it & 1)), 0));
      }
      if (!ok) break;
      // a barrier of its own: o_done may be two phases behind here
      wait(o_last, pieces & 1);
      ++pieces;
      if (!ok) break;
      tc_fence_after();
      const bool whole = w.j0 == 0 && w.j1 == w.nb;
      const int place = pair * 2 + (w.j0 == 0 ? 1 : 0), row = (int)rank * 128 + rr;
      if (!whole) {
        ws.ml[((size_t)place * 256 + row) * 2] = m;
        ws.ml[((size_t)place * 256 + row) * 2 + 1] = l;
        if (w.j0 == 0) {
          // the part that holds the tile's last block
          const long long u = work.begin + work.count + (w.nb - w.j1) - 1, g = min((long long)pairs, work.total);
          desc = make_int4(w.b, w.head, w.tile, (int)(((u + 1) * g - 1) / work.total));
        }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      T* dst = static_cast<T*>(p.out) + (long long)(w.s.q0 + tok) * p.out_token +
               (long long)(w.head * p.group + hd) * p.out_head;
      float* wo = ws.o + ((size_t)place * 256 + row) * D;
#pragma unroll 1
      for (int i = 0; i < D / 32; ++i) {
        float o[32];
        tmem_ld32(lanes + C::COL_O + 32 * i, o);
        tmem_ld_wait();
        if (whole && row_ok) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4 u;
            u.x = Elem<T>::from_f2(o[8 * q] * inv, o[8 * q + 1] * inv);
            u.y = Elem<T>::from_f2(o[8 * q + 2] * inv, o[8 * q + 3] * inv);
            u.z = Elem<T>::from_f2(o[8 * q + 4] * inv, o[8 * q + 5] * inv);
            u.w = Elem<T>::from_f2(o[8 * q + 6] * inv, o[8 * q + 7] * inv);
            if (l <= 0.f) u = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(dst + 32 * i + 8 * q) = u;
          }
        } else if (row_ok) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(wo + 32 * i + 4 * q) =
                make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(o_free), 0));
    }
    if (rank == 0 && tid == 0) ws.desc[pair] = desc;
  } else if (E4) {
    // ---- codes: warps 6-9 load, widen and store this CTA's halves
    const int t = tid - 192;
    constexpr int PIECES = 64 * D / 16 / 128;      // 16-code pieces of a thread
    int slot = 0;
    uint32_t phase = 0, kn = 0;
    bool ok = true;
    auto load = [&](const ChunkPiece& x, int j, bool is_v) {
      // K: 64 keys x D; V: 128 keys x D/2
      const int per_row = is_v ? D / 32 : D / 16;
      uint4 u[PIECES];
      float sc[PIECES];
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int at = i * 128 + t, r = at / per_row, c = at - r * per_row;
        const int key = j * kBlockKeys + (is_v ? 0 : 64 * (int)rank) + r;
        u[i] = make_uint4(0, 0, 0, 0);
        sc[i] = 0.f;
        if (key < x.s.kv) {
          const int id = __ldcg(p.table + (long long)x.b * p.table_stride + (key >> p.page_shift));
          if (id >= 0 && id < p.pages) {
            const long long row = ((long long)(id * p.kv_heads + x.head) << p.page_shift) + (key & (ps - 1));
            u[i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(is_v ? p.v_codes : p.k_codes) +
                                                         row * D + (is_v ? (int)rank * (D / 2) : 0) + c * 16));
            if (is_v) sc[i] = __ldcg(p.v_scale + row);
          }
        }
      }
      float ks = 0.f;
      if (!is_v) {
        // both CTAs need the scales of all 128 keys
        const int key = j * kBlockKeys + t;
        if (key < x.s.kv) {
          const int id = __ldcg(p.table + (long long)x.b * p.table_stride + (key >> p.page_shift));
          if (id >= 0 && id < p.pages)
            ks = __ldcg(p.k_scale + ((long long)(id * p.kv_heads + x.head) << p.page_shift) + (key & (ps - 1)));
        }
      }
      if (ok && !mbar_wait(empty + slot, phase ^ 1, kAttnWaitBudgetNs)) {
        if (lane == 0) attn_error(p.err, kAttnErrChunkWiden);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok && !s_abort);
      if (!ok) return;
      uint8_t* dst = smem + C::Q_BYTES + (size_t)slot * C::SLOT;
      const int rows = is_v ? kBlockKeys : 64;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int at = i * 128 + t, r = at / per_row, c = at - r * per_row;
        const uint32_t w4[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        uint32_t o[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (is_v) {
            o[2 * q] = widen2<T>((uint16_t)w4[q], sc[i]);
            o[2 * q + 1] = widen2<T>((uint16_t)(w4[q] >> 16), sc[i]);
          } else {
            o[2 * q] = widen2<T>((uint16_t)w4[q]);
            o[2 * q + 1] = widen2<T>((uint16_t)(w4[q] >> 16));
          }
        }
        // 16 values: two 16-byte pieces of a 64-dim column
        uint8_t* col = dst + (c >> 2) * (rows * 128) + r * 128;
        const int pc = (c & 3) * 2;
        *reinterpret_cast<uint4*>(col + (((pc ^ r) & 7) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(col + ((((pc + 1) ^ r) & 7) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      if (!is_v) {
        s_ks[(kn % C::KS_RING) * kBlockKeys + t] = ks;
        ++kn;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa(smem_u32(full + slot), 0));
      if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
    };
    while (ok && walk.next(p, per, w)) {
      for (int j = w.j0; j < w.j1 && ok; ++j) {
        load(w, j, false);
        if (j > w.j0 && ok) load(w, j - 1, true);
      }
      if (ok) load(w, w.j1 - 1, true);
    }
    if (!ok) s_abort = 1;
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // every MMA of the pair, and every arrival that it makes here, has ended
  // before TMEM or shared memory goes
  if (warp == 4 && !mbar_wait_cluster(all_done, 0) && lane == 0) attn_error(p.err, kAttnErrChunkMma);
  __syncwarp();
  cluster_sync_all();      // no CTA leaves while its pair may still arrive at it
  tc_fence_after();
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Tiles that the parts' cuts go through: the sum of their parts, in order.
// blockIdx.x is the part in which the tile begins, blockIdx.y a group of rows.
constexpr int kJoinRows = 16;
template <typename T, int D>
__global__ void __launch_bounds__(256) attn_chunk_join_kernel(const __grid_constant__ AttnParams p, const ChunkWs ws) {
  pdl_trigger();
  pdl_wait();
  const int c0 = blockIdx.x;
  const int4 de = __ldcg(ws.desc + c0);
  if (de.w < 0) return;
  const int b = de.x, head = de.y, tile = de.z, c1 = de.w;
  const AttnSeq s = attn_seq(p, b);
  const int tpc = 128 / p.group;
  for (int i = threadIdx.x; i < kJoinRows * (D / 4); i += 256) {
    const int row = blockIdx.y * kJoinRows + i / (D / 4), d = (i % (D / 4)) * 4;
    const int rr = row & 127, ti = rr / p.group, tok = tile * 2 * tpc + (row >> 7) * tpc + ti;
    if (ti >= tpc || tok >= s.n) continue;
    float m = -INFINITY;
    for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(ws.ml + (((size_t)c * 2 + (c == c0)) * 256 + row) * 2));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const size_t at = ((size_t)c * 2 + (c == c0)) * 256 + row;
      const float mc = __ldcg(ws.ml + at * 2);
      if (mc == -INFINITY) continue;
      const float f = ex2(mc - m);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(ws.o + at * D + d));
      l = fmaf(__ldcg(ws.ml + at * 2 + 1), f, l);
      a.x = fmaf(v.x, f, a.x);
      a.y = fmaf(v.y, f, a.y);
      a.z = fmaf(v.z, f, a.z);
      a.w = fmaf(v.w, f, a.w);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* dst = static_cast<T*>(p.out) + (long long)(s.q0 + tok) * p.out_token +
             (long long)(head * p.group + rr - ti * p.group) * p.out_head + d;
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(Elem<T>::from_f2(a.x * inv, a.y * inv), Elem<T>::from_f2(a.z * inv, a.w * inv));
  }
}

}  // namespace d3
