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
// for the exponentials of 128 x 128 scores on one warpgroup), the exponentials
// for D = 128.  Measured, 2048 tokens over 14000, pages of 64: 16 heads of 256
// over 2 in bf16 1425 TFLOP/s, 32 of 128 over 8 in fp16 983; the former, run for
// seconds, is held by the power limit.  Pages of 16 hold 16-bit caches back
// (1095 and 635): their loading threads issue many small boxes a block.
// Codes reach 860 and 560, bound by instruction-cache misses (six of ten
// cycles issue nothing): the widening and the softmax are different code on
// the same schedulers, which is why their loops are kept short.
//
// TMEM, 512 columns: two S blocks (P of each half goes over its S) and O.  S of block
// j + 1 is issued before P V of block j, so the tensor core works while the
// softmax does.  O is only rescaled when a row's maximum grows by more than 8
// (in log2): P then stays below 2^8, sums are in fp32 and the quotient of the
// two does not change.
//
// Roles (per CTA): warps 0-7 softmax and output (a row is shared by two
// threads, 64 keys of a block and half of O each), warp 8 issues the MMAs (in
// the pair's first CTA), one thread each of warps 9 and 10 the TMA loads of Q
// and K and of V; for codes warp 11 brings the scales and warps 12-15 widen
// the tiles.
//
// A block's last page, when the sequence ends in it, is loaded shifted: rows
// before the page's first come from outside the tensor map and are zeros, the
// page's valid rows follow, and what lies behind the end (NaN, perhaps) never
// reaches shared memory.  The mask knows about the shift.
//
// Split: as in the row kernel, the list of all (sequence, KV head, row tile,
// key block) is cut into equal parts, one per pair; tiles that a cut goes
// through are joined by attn_join_kernel in the parts' order.
//
// e4m3 caches: codes are staged by TMA and widened to 16 bits in shared
// memory.  K codes are exact there, and a key's scale multiplies a column of S
// in fp32.  A value's scale is split into 2^e, by which the widened codes are
// multiplied (exact again), and f in [1, 2), which multiplies a column of P in
// fp32 before P is rounded: one rounding on the way, as with a 16-bit cache.
#pragma once

#include "attn_rows.cuh"

namespace d3 {

constexpr int kAttnErrChunkLoad = 53, kAttnErrChunkMma = 54, kAttnErrChunkSoftmax = 55,
              kAttnErrChunkWiden = 56, kAttnErrChunkAlign = 57;
constexpr int kBlockKeys = 128;
constexpr float kRescaleLog2 = 8.f;
// Pages below this go into the code ring by 16-byte copies of a whole warp: a
// TMA instruction costs its thread some 500 cycles here whatever its size.
// 2048 tokens over 14000, 8 heads x 128: pages of 16 take 1204 us by TMA and
// 990 by copies, of 32 1081 and 912, of 64 996 and 901, but of 128, one
// instruction a tile, 801 and 902.
constexpr int kSmallPage = 128;

template <typename T, int D, bool E4>
struct ChunkCfg {
  static constexpr int THREADS = E4 ? 512 : 352;
  static constexpr int Q_BYTES = 128 * D * 2;
  static constexpr int SLOT = 64 * D * 2;                 // half a block of K or of V
  static constexpr int SLOTS = E4 ? (D == 256 ? 3 : 6) : (D == 256 ? 5 : 10);
  static constexpr int RAW = E4 ? 64 * D : 0;             // the same as codes
  static constexpr int RAWS = E4 ? (D == 256 ? 3 : 6) : 0;
  static constexpr int SC_RING = 4;                       // scales of 4 blocks: ks, f, 2^e in two words
  static constexpr int SC_BYTES = E4 ? SC_RING * 4 * kBlockKeys * 4 : 0;
  static constexpr size_t SMEM =
      1024 + Q_BYTES + (size_t)SLOTS * SLOT + (size_t)RAWS * RAW + SC_BYTES + 2048 + (E4 ? 256 : 0);
  static constexpr int COL_S = 0, COL_O = 256;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct ChunkWs {           // carved from the call's workspace
  float* o;                // [pairs][2][D / 4][256][4]
  float* ml;               // [pairs][2][256][2]
  int4* desc;              // [pairs][2]: (first query token, new tokens, KV head, row tile), (last part or -1,
                           // last key of the sequence's first new token, ...)
};

// key blocks that row tile i (of `per` tokens) of a sequence sees: at least one
__device__ __forceinline__ int chunk_blocks(const AttnSeq& s, int per, int i) {
  const int vis = s.kv - s.n + min((i + 1) * per, s.n);
  return max(1, (vis + kBlockKeys - 1) / kBlockKeys);
}
__device__ __forceinline__ int chunk_tiles(const AttnSeq& s, int per) { return (s.n + per - 1) / per; }
__device__ __forceinline__ bool chunk_takes(const AttnParams& p, const AttnSeq& s) {
  return s.rows > 0 && s.rows >= p.min_rows && s.rows <= p.max_rows;
}
__device__ __forceinline__ AttnSeq seq_from(const AttnSeq& s, int lane) {
  AttnSeq r;
  r.q0 = __shfl_sync(0xffffffffu, s.q0, lane);
  r.n = __shfl_sync(0xffffffffu, s.n, lane);
  r.kv = __shfl_sync(0xffffffffu, s.kv, lane);
  r.rows = __shfl_sync(0xffffffffu, s.rows, lane);
  return r;
}
// Every row tile stands in the list with its key blocks and `more` units in
// front of them, about what a piece costs besides (queries in, output out): a
// prompt's first tiles have one block each.
template <int D>
constexpr int kTileUnits = D == 256 ? 2 : 3;
// one warp: units of all row tiles of a sequence, for one KV head
__device__ __forceinline__ int warp_head_units(const AttnSeq& s, int per, int more) {
  int u = 0;
  for (int i = threadIdx.x & 31; i < chunk_tiles(s, per); i += 32) u += chunk_blocks(s, per, i) + more;
  return __reduce_add_sync(0xffffffffu, u);
}

// A part of the list: where it begins and how long it is.
struct ChunkPart {
  int total, begin, count;
  int b, head, tile, pos;        // place in the tile's units
  AttnSeq s;
};
// All threads of the CTA.  Each warp takes a run of sequences, 32 at a time:
// their lanes read the lengths, and the whole warp adds up the blocks of each
// that this launch takes.
__device__ ChunkPart chunk_plan(const AttnParams& p, int per, int more, int part, int parts, int* s_scan,
                                ChunkPart* s_part) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = (p.batch + warps - 1) / warps, b0 = min(p.batch, warp * run), b1 = min(p.batch, b0 + run);
  int sum = 0;
  AttnSeq held{0, 0, 0, 0};      // the lane's first sequence, read once
  if (b0 + lane < b1) held = attn_seq(p, b0 + lane);
  auto each = [&](auto f) {      // f(b, sequence) until it says true
    for (int at = b0; at < b1; at += 32) {
      AttnSeq s = held;
      if (at > b0 && at + lane < b1) s = attn_seq(p, at + lane);
      unsigned todo = __ballot_sync(0xffffffffu, at + lane < b1 && chunk_takes(p, s));
      while (todo) {
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        if (f(at + i, seq_from(s, i))) return;
      }
    }
  };
  each([&](int, const AttnSeq& s) {
    sum = list_add(sum, warp_head_units(s, per, more) * p.kv_heads);
    return false;
  });
  if (lane == 0) s_scan[warp] = sum;
  __syncthreads();
  int before = 0, total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before = list_add(before, s_scan[w]);
    total = list_add(total, s_scan[w]);
  }
  total = list_total(p, total);
  const int g = min(parts, total);
  const int begin = part < g ? part_begin(total, g, part) : 0;
  const int count = part < g ? part_begin(total, g, part + 1) - begin : 0;
  if (count > 0 && before <= begin && begin < before + sum) {
    int at = before;
    each([&](int b, const AttnSeq& s) {
      const int u = warp_head_units(s, per, more);
      if (begin >= at + u * p.kv_heads) {
        at += u * p.kv_heads;
        return false;
      }
      const int head = (begin - at) / u;
      int r = begin - at - head * u;
      for (int i0 = 0;; i0 += 32) {          // the row tile: 32 at a time
        const int i = i0 + lane;
        const int n = i < chunk_tiles(s, per) ? chunk_blocks(s, per, i) + more : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        const int all = __shfl_sync(0xffffffffu, inc, 31);
        if (r < all) {
          if (inc - n <= r && r < inc) *s_part = ChunkPart{total, begin, count, b, head, i, r - (inc - n), s};
          return true;
        }
        r -= all;
      }
    });
  } else if (count == 0 && threadIdx.x == 0) {
    *s_part = ChunkPart{total, 0, 0, 0, 0, 0, 0, {0, 0, 0, 0}};
  }
  __syncthreads();
  return *s_part;
}

struct ChunkHead {         // the first 1024 bytes of shared memory
  uint64_t bars[64];
  int scan[16];
  ChunkPart part;
  uint32_t tmem;
  int abort;
};

struct ChunkPiece {
  AttnSeq s;
  int b, head, tile, j0, j1, nb;
};
// Walks a part piece by piece.
struct ChunkWalk {
  int b, left, head, tile, pos, more;
  bool fresh;
  AttnSeq s;
  __device__ __forceinline__ ChunkWalk(const ChunkPart& c, int more_)
      : b(c.b), left(c.count), head(c.head), tile(c.tile), pos(c.pos), more(more_), fresh(true), s(c.s) {}
  __device__ __forceinline__ bool next(const AttnParams& p, int per, ChunkPiece& w) {
    while (left > 0) {
      if (fresh) {
        fresh = false;
      } else {
        pos = 0;
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
      const int nb = chunk_blocks(s, per, tile), take = min(left, nb + more - pos);
      left -= take;
      w.s = s;
      w.b = b;
      w.head = head;
      w.tile = tile;
      w.nb = nb;
      w.j0 = max(0, pos - more);
      w.j1 = max(0, pos + take - more);
      if (w.j1 > w.j0) return true;      // else nothing but the units in front
    }
    return false;
  }
};
// Walks it tile by tile in the order of the ring: K j0, K j0 + 1, V j0, ...,
// K last, V last - 1, V last.
struct ChunkTiles {
  ChunkWalk walk;
  ChunkPiece w;
  int j, step;
  bool is_v;
  __device__ __forceinline__ ChunkTiles(const ChunkPart& c, int more) : walk(c, more), step(-1) { w.j0 = w.j1 = 0; }
  __device__ __forceinline__ bool next(const AttnParams& p, int per) {
    // steps of a piece of n blocks: 0: K0; 2k - 1: K k; 2k: V k - 1; 2n - 1: V n - 1
    const int n = w.j1 - w.j0;
    if (step < 0 || ++step >= 2 * n) {
      if (!walk.next(p, per, w)) return false;
      step = 0;
    }
    const int m = w.j1 - w.j0;
    is_v = step == 2 * m - 1 || (step > 0 && (step & 1) == 0);
    j = w.j0 + (step == 2 * m - 1 ? m - 1 : is_v ? step / 2 - 1 : (step + 1) / 2);
    return true;
  }
};
// A warp's window of a sequence's page table: 32 entries in the lanes, the 32
// behind them on their way.  A look-up of each tile's pages would cost the
// loading warp an L2 round trip a tile, about as long as the tile's MMAs.
struct PageWindow {
  int b, base, now, then;
  __device__ __forceinline__ PageWindow() : b(-1), base(0), now(0), then(0) {}
  __device__ __forceinline__ int fetch(const AttnParams& p, int pg) const {
    return pg < p.table_pages ? __ldcg(p.table + (long long)b * p.table_stride + pg) : -1;
  }
  // all lanes: makes the pages of the key block that begins at page pg of
  // sequence nb available.  Blocks come in order, but for V of the block
  // before the last K: a slide keeps that one.
  __device__ __forceinline__ void reach(const AttnParams& p, int nb, int pg) {
    const int lane = threadIdx.x & 31, need = kBlockKeys >> p.page_shift;
    if (nb == b && pg >= base && pg + need <= base + 32) return;
    if (nb == b && pg == base + 32) {
      const int lo = __shfl_sync(0xffffffffu, now, (lane + 32 - need) & 31);
      const int hi = __shfl_sync(0xffffffffu, then, (lane - need) & 31);
      now = lane < need ? lo : hi;
      base = pg - need;
    } else {
      b = nb;
      base = pg;
      now = fetch(p, pg + lane);
    }
    then = fetch(p, base + 32 + lane);
  }
  // all lanes: where row `key` of the sequence lies: its page, as a plane of
  // the tensor map (-1: none), and the row inside it.  The sequence's last
  // page is read late by what it lacks, so that its valid rows come last.
  __device__ __forceinline__ void row(const AttnParams& p, const ChunkPiece& w, int key, int& plane, int& row) const {
    const int pg = key >> p.page_shift, start = pg << p.page_shift;
    const int id = __shfl_sync(0xffffffffu, now, (pg - base) & 31);
    plane = start < w.s.kv && id >= 0 && id < p.pages ? id * p.kv_heads + w.head : -1;
    row = key - start - max(0, start + p.page_size - w.s.kv);
  }
};

// One thread's walk of a part block by block, a block ahead of what it loads:
// the page ids of the next block are on their way while this one's TMA
// instructions go out.  (An L2 round trip, or the shuffles and votes of a
// whole warp, for every tile cost as much as the tile's MMAs.)
struct ChunkBlocks {
  ChunkWalk walk;
  ChunkPiece w;
  int j;
  bool more;
  int ids[8];
  __device__ __forceinline__ ChunkBlocks(const ChunkPart& c, int units) : walk(c, units), j(0), more(false) {}
  __device__ __forceinline__ void fetch(const AttnParams& p, int key0, int box, int n) {
    const int* row = p.table + (long long)w.b * p.table_stride;
    const int key = j * kBlockKeys + key0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) {
        const int pg = (key + i * box) >> p.page_shift;
        ids[i] = (pg << p.page_shift) < w.s.kv ? __ldcg(row + pg) : -1;
      }
  }
  __device__ __forceinline__ void first(const AttnParams& p, int per, int key0, int box, int n) {
    more = walk.next(p, per, w);
    if (!more) return;
    j = w.j0;
    fetch(p, key0, box, n);
  }
  __device__ __forceinline__ void step(const AttnParams& p, int per, int key0, int box, int n) {
    if (++j >= w.j1) {
      more = walk.next(p, per, w);
      if (!more) return;
      j = w.j0;
    }
    fetch(p, key0, box, n);
  }
};
// Where `key` of a sequence with page id `id` lies: plane of the tensor map
// (-1: none) and row of the page.  The sequence's last page is read late by
// what it lacks, so that its valid rows come last.
__device__ __forceinline__ void page_place(const AttnParams& p, int id, int head, int kv, int key, int& plane, int& row) {
  const int start = key & -p.page_size;
  plane = id >= 0 && id < p.pages ? id * p.kv_heads + head : -1;
  row = key - start - max(0, start + p.page_size - kv);
}
// A place in a ring of n slots, moved on by up to n.
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance(int d, int n) {
    slot += d;
    if (slot >= n) {
      slot -= n;
      phase ^= 1;
    }
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
// an arrival at a barrier of either CTA.  What it publishes is in shared memory
// or TMEM of this CTA; a release of cluster scope would also wait for the
// thread's global stores, which cost 1300 cycles a block.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// loads of a pair's CTA that complete on a barrier of either CTA; no multicast
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x),
      "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_pair_4d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z, int u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x),
      "r"(y), "r"(z), "r"(u)
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
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t* u) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(u[0]), "r"(u[1]),
               "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t a, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(a));
}
__device__ __forceinline__ void tmem_st4(uint32_t a, const uint32_t* u) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(u[0]), "r"(u[1]), "r"(u[2]),
               "r"(u[3])
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
// ... times a power of two: two fp16 factors, or one fp32 one
template <typename T>
__device__ __forceinline__ uint32_t widen2(uint16_t c, uint32_t ea, uint32_t eb);
template <>
__device__ __forceinline__ uint32_t widen2<__half>(uint16_t c, uint32_t ea, uint32_t eb) {
  const uint32_t h = e4m3x2_to_h2(c);
  __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&ea));
  x = __hmul2(x, *reinterpret_cast<const __half2*>(&eb));
  return *reinterpret_cast<const uint32_t*>(&x);
}
template <>
__device__ __forceinline__ uint32_t widen2<__nv_bfloat16>(uint16_t c, uint32_t ea, uint32_t) {
  float2 f = e4m3x2_to_f2(c);
  mul2(f.x, f.y, __uint_as_float(ea), __uint_as_float(ea));
  return Elem<__nv_bfloat16>::from_f2(f.x, f.y);
}

// ---------------------------------------------------------------- kernel

template <typename T, int D, bool E4>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ChunkCfg<T, D, E4>::THREADS, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnParams p,
                      const ChunkWs ws) {
  using C = ChunkCfg<T, D, E4>;
  constexpr int MORE = kTileUnits<D>;
  // no static shared memory: the dynamic part begins on a 1024-byte boundary
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  ChunkHead& head = *reinterpret_cast<ChunkHead*>(smem_raw);
  static_assert(sizeof(ChunkHead) <= 1024, "head of shared memory");
  volatile int& s_abort = head.abort;
  uint8_t* smem = smem_raw + 1024;
  uint8_t* at = smem + C::Q_BYTES;
  uint8_t* s_ring = at;
  at += (size_t)C::SLOTS * C::SLOT;
  uint8_t* s_codes = at;
  at += (size_t)C::RAWS * C::RAW;
  float* s_sc = reinterpret_cast<float*>(at);           // [SC_RING][ks, f, 2^e, 2^e][128]
  at += C::SC_BYTES;
  float* s_mx = reinterpret_cast<float*>(at);           // [2][2][128]
  float* s_one = s_mx + 512;                            // [64] ones
  uint64_t* full = head.bars;
  uint64_t* empty = full + C::SLOTS;
  uint64_t* q_full = empty + C::SLOTS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;        // [2]
  uint64_t* p_ready = s_full + 2;        // [2]
  uint64_t* o_done = p_ready + 2;
  uint64_t* o_free = o_done + 1;
  uint64_t* o_last = o_free + 1;
  uint64_t* all_done = o_last + 1;
  uint64_t* raw_full = all_done + 1;     // codes: [RAWS]
  uint64_t* raw_empty = raw_full + C::RAWS;
  uint64_t* sc_full = raw_empty + C::RAWS;   // [SC_RING]
  uint64_t* sc_empty = sc_full + C::SC_RING;
  static_assert(2 * C::SLOTS + 10 + 2 * C::RAWS + 2 * C::SC_RING <= 64, "barriers");
  const uint32_t sq = smem_u32(smem), ss = smem_u32(s_ring);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int ps = p.page_size;
  if (smem_u32(smem_raw) & 1023) {       // the swizzle counts on it
    if (tid == 0) {
      attn_error(p.err, kAttnErrChunkAlign);
      ws.desc[blockIdx.x | 1] = make_int4(-1, 0, 0, 0);      // nothing to join
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, E4 ? 8 : 1);   // codes: four widening warps of either CTA
      mbar_init(empty + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 16);        // eight warps of either CTA
    }
    mbar_init(o_done, 1);
    mbar_init(o_free, 16);
    mbar_init(o_last, 1);
    mbar_init(all_done, 1);
    if (E4) {
      for (int i = 0; i < C::RAWS; ++i) {
        mbar_init(raw_full + i, ps < kSmallPage ? 32 : 1);     // 32 lanes' copies, or TMA
        mbar_init(raw_empty + i, 4);
      }
      for (int i = 0; i < C::SC_RING; ++i) {
        mbar_init(sc_full + i, 1);
        mbar_init(sc_empty + i, 12);     // eight softmax, four widening warps
      }
    }
    fence_barrier_init();
    s_abort = 0;
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (E4 && tid >= 128 && tid < 192) s_one[tid - 128] = 1.f;
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&head.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = head.tmem;
  pdl_trigger();
  if (!p.beside) pdl_wait();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tpc = 128 / p.group, per = 2 * tpc;      // tokens of a CTA, of the pair
  const ChunkPart part = chunk_plan(p, per, MORE, pair, pairs, head.scan, &head.part);
  cluster_sync_all();      // both CTAs' barriers are ready

  bool ok = true;
  // every lane of a warp: false once a wait has run out, here or in another role
  auto wait_warp = [&](uint64_t* bar, uint32_t par, int code) {
    if (ok && !__all_sync(0xffffffffu, mbar_try_wait(bar, par)))
      ok = __all_sync(0xffffffffu, wait_on(smem_u32(bar), par, p.err, code, &s_abort));
    return ok;
  };
  // one thread
  auto wait_one = [&](uint64_t* bar, uint32_t par, int code) {
    if (ok && !mbar_try_wait(bar, par)) ok = wait_on(smem_u32(bar), par, p.err, code, &s_abort);
    return ok;
  };

  // Q of a piece (one thread): rows (token, head) of both CTAs
  auto load_q = [&](const ChunkPiece& x) {
    if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * (D / 64) * tpc * p.group * 128);
    const uint32_t bar = mapa(smem_u32(q_full), 0);
    const int tok = x.s.q0 + x.tile * per + (int)rank * tpc;
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) tma_pair_3d(sq + c * (128 * 128), &tm_q, bar, c * 64, x.head * p.group, tok);
  };

  if (E4 && ps < kSmallPage && (warp == 9 || warp == 10)) {
    // ---- codes of small pages: a warp copies K, one V, as the TMA threads
    // below would (same ring, same shifted last page), 512 bytes an instruction
    auto copy = [&](auto is_v) {
      constexpr bool v = decltype(is_v)::value;
      constexpr int RB = v ? D / 2 : D, PPR = RB / 16, RPI = 32 / PPR, ROWS = v ? kBlockKeys : 64;
      const uint8_t* src0 = static_cast<const uint8_t*>(v ? p.v_codes : p.k_codes) + (v ? (int)rank * RB : 0) +
                            (lane % PPR) * 16;
      const int n = ROWS / ps, half = v ? 0 : 64 * (int)rank;
      ChunkWalk walk(part, MORE);
      ChunkPiece x;
      bool more = walk.next(p, per, x);
      int j = more ? x.j0 : 0, id_next = -1, at_pos = 0, base = 0;
      uint32_t qn = 0;
      RingPos pos;
      auto fetch = [&]() {       // lane i: page i of the tile, a block ahead
        const int key = j * kBlockKeys + half + lane * ps;
        id_next = lane < n && key < x.s.kv ? __ldcg(p.table + (long long)x.b * p.table_stride + (key >> p.page_shift)) : -1;
      };
      if (more) fetch();
      while (more) {
        const ChunkPiece y = x;
        const int key0 = j * kBlockKeys + half, m = x.j1 - x.j0, k = j - x.j0;
        const int plane = id_next >= 0 && id_next < p.pages ? id_next * p.kv_heads + x.head : -1;
        if (++j >= x.j1) {
          more = walk.next(p, per, x);
          j = more ? x.j0 : 0;
        }
        if (more) fetch();
        const int want = base + (v ? (k == m - 1 ? 2 * m - 1 : 2 * k + 2) : (k ? 2 * k - 1 : 0));
        for (; at_pos < want; ++at_pos) pos.advance(1, C::RAWS);
        if (k == m - 1) base += 2 * m;
        if (!v && k == 0) {
          if (!wait_warp(q_empty, (qn & 1) ^ 1, kAttnErrChunkLoad)) break;
          ++qn;
          if (lane == 0) load_q(y);
          __syncwarp();
        }
        if (!wait_warp(raw_empty + pos.slot, pos.phase ^ 1, kAttnErrChunkLoad)) break;
        uint32_t dst = smem_u32(s_codes) + pos.slot * C::RAW + lane * 16;
        for (int pg = 0; pg < n; ++pg) {
          const int pl = __shfl_sync(0xffffffffu, plane, pg);
          const int row = lane / PPR - max(0, key0 + pg * ps + ps - y.s.kv);
          const uint8_t* src = src0 + (((long long)pl << p.page_shift) + row) * D;
#pragma unroll 4
          for (int i = 0; i < ps; i += RPI) {
            const bool in = pl >= 0 && row + i >= 0;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? src + i * D : src0), "r"(in ? 16 : 0)
                         : "memory");
            dst += 512;
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(raw_full + pos.slot)) : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      // after a wait ran out: Q, too, has landed before the memory goes
      if (!ok && qn && rank == 0) mbar_wait(q_full, (qn - 1) & 1, kAttnWaitBudgetNs);
    };
    if (warp == 9) copy(std::false_type{});
    else copy(std::true_type{});
  } else if (warp == 9 || warp == 10) {
    // ---- TMA: one thread brings Q of a piece and its K tiles, one its V
    // tiles.  The tiles of a piece of m blocks stand in the ring as K 0, K 1,
    // V 0, K 2, V 1, ..., K m - 1, V m - 2, V m - 1.
    if (lane == 0) {
      constexpr int N = E4 ? C::RAWS : C::SLOTS;
      uint64_t* bars_full = E4 ? raw_full : full;
      uint64_t* bars_empty = E4 ? raw_empty : empty;
      RingPos pos;
      const bool v = warp == 10;
      // One box a page with all of its columns of 64 dims, but for 16-bit K of
      // small pages, whose rows of one column have to lie together.
      const int rows = v ? kBlockKeys : 64, box = min(ps, rows), n = rows / box;
      const int key0 = v ? 0 : 64 * (int)rank;
      ChunkBlocks bl(part, MORE);
      bl.first(p, per, key0, box, n);
      uint32_t qn = 0;
      int at_pos = 0, base = 0;
      while (bl.more) {
        const ChunkPiece x = bl.w;
        const int j = bl.j, m = x.j1 - x.j0, k = j - x.j0;
        int ids[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) ids[i] = bl.ids[i];
        bl.step(p, per, key0, box, n);
        const int want = base + (v ? (k == m - 1 ? 2 * m - 1 : 2 * k + 2) : (k ? 2 * k - 1 : 0));
        for (; at_pos < want; ++at_pos) pos.advance(1, N);
        if (k == m - 1) base += 2 * m;
        if (!v && k == 0) {
          if (!wait_one(q_empty, (qn & 1) ^ 1, kAttnErrChunkLoad)) break;
          ++qn;
          load_q(x);
        }
        if (!wait_one(bars_empty + pos.slot, pos.phase ^ 1, kAttnErrChunkLoad)) break;
        if (E4) mbar_arrive_expect_tx(bars_full + pos.slot, C::RAW);
        else if (rank == 0) mbar_arrive_expect_tx(bars_full + pos.slot, 2 * C::SLOT);
        const uint32_t bar = E4 ? smem_u32(bars_full + pos.slot) : mapa(smem_u32(bars_full + pos.slot), 0);
        const uint32_t dst = E4 ? smem_u32(s_codes) + pos.slot * C::RAW : ss + pos.slot * C::SLOT;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < n) {
            int y, u;
            page_place(p, ids[i], x.head, x.s.kv, j * kBlockKeys + key0 + i * box, u, y);
            if (E4) {
              if (v) tma_load_4d(dst + i * box * (D / 2), &tm_v, bar, (int)rank * (D / 2), y, 0, u);
              else tma_load_4d(dst + i * box * D, &tm_k, bar, 0, y, 0, u);
            } else if (v) {
              tma_pair_4d(dst + i * box * D, &tm_v, bar, 0, y, (int)rank * (D / 128), u);
            } else if (n == 1) {
              tma_pair_4d(dst, &tm_k, bar, 0, y, 0, u);
            } else {
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
                tma_pair_4d(dst + c * (64 * 128) + i * (box * 128), &tm_k, bar, 0, y, c, u);
            }
          }
        }
      }
      // after a wait ran out: what is in flight has landed before the memory goes
      if (!ok && (E4 || rank == 0))
        drain_ring(N, pos.slot, pos.phase, kAttnWaitBudgetNs,
                   [&](int i, uint32_t par) { return mbar_try_wait(bars_full + i, par); },
                   [] { return globaltimer_ns(); });
      if (!ok && qn && rank == 0) mbar_wait(q_full, (qn - 1) & 1, kAttnWaitBudgetNs);
    }
  } else if (warp == 8) {
    // ---- MMAs of the pair
    if (rank == 0 && lane == 0) {
      constexpr uint32_t id_s = idesc_16<T>(256, kBlockKeys, false), id_o = idesc_16<T>(256, D, true);
      ChunkWalk walk(part, MORE);
      ChunkPiece w;
      int slot = 0;
      uint32_t phase = 0, it = 0, pieces = 0;
      // V: pages of `vrows` keys, each [D / 128 columns][vrows][128 bytes]; 16 keys a k-step
      const int vrows = E4 ? kBlockKeys : ps;
      const uint64_t qd = smem_desc_k128(sq);
      auto wait = [&](uint64_t* bar, uint32_t par) { return wait_one(bar, par, kAttnErrChunkMma); };
      auto advance = [&]() {
        commit_pair(empty + slot);
        if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
      };
      auto scores = [&](uint32_t x) {
        if (!wait(full + slot, phase)) return;
        tc_fence_after();
        // descriptors count in 16 bytes: a k-step is an addition
        const uint64_t kd = smem_desc_k128(ss + slot * C::SLOT);
        const uint32_t d = tmem + C::COL_S + (x & 1) * kBlockKeys;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_pair_ss(d, qd + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16,
                      kd + ((k >> 2) * (64 * 128) + (k & 3) * 32) / 16, id_s, k > 0);
        commit_pair(s_full + (x & 1));
        advance();
      };
      auto values = [&](uint32_t x, bool first) {
        if (!wait(full + slot, phase)) return;
        if (!wait(p_ready + (x & 1), (x >> 1) & 1)) return;
        if (first && pieces > 0 && !wait(o_free, (pieces - 1) & 1)) return;
        tc_fence_after();
        const uint64_t vd = smem_desc_n128(ss + slot * C::SLOT, vrows * 128);
        const uint32_t a = tmem + C::COL_S + (x & 1) * kBlockKeys;
#pragma unroll
        for (int k = 0; k < kBlockKeys / 16; ++k)
          mma_pair_ts(tmem + C::COL_O, a + (k >> 2) * 64 + (k & 3) * 8,
                      vd + ((k * 16 & -vrows) * D + (k * 16 & (vrows - 1)) * 128) / 16, id_o, !first || k > 0);
        commit_pair(o_done);
        advance();
      };
      while (ok && walk.next(p, per, w)) {
        if (!wait(q_full, pieces & 1)) break;
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
  } else if (warp < 8) {
    // ---- softmax: a row's thread of half h has keys [64 h, 64 h + 64) of a
    // block and dims [h D/2, (h + 1) D/2) of the output
    const int h = warp >> 2, quarter = warp & 3, rr = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t mine_o = lanes + C::COL_O + h * (D / 2);
    const int ti = rr / p.group, hd = rr - ti * p.group;
    // the value that the row's other thread gives.  Two buffers: a thread is
    // one exchange ahead at most.  The barrier among the row's two warps is
    // safe because both always come: after a wait has run out the loops go on
    // to their end without waiting.
    uint32_t xn = 0;
    auto exchange = [&](float v) {
      float* buf = s_mx + (xn++ & 1) * 256 + rr;
      buf[h * 128] = v;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
      return buf[(h ^ 1) * 128];
    };
    auto wait = [&](uint64_t* bar, uint32_t par) { wait_warp(bar, par, kAttnErrChunkSoftmax); };
    ChunkWalk walk(part, MORE);
    ChunkPiece w{};
    uint32_t it = 0, pieces = 0;
    const float c = p.scale_log2;
    while (walk.next(p, per, w)) {
      const int tok = w.tile * per + (int)rank * tpc + ti;       // of the sequence's new ones
      const bool row_ok = ti < tpc && tok < w.s.n;
      const int last = row_ok ? w.s.kv - w.s.n + tok : 1 << 30;
      const bool idle = !__any_sync(0xffffffffu, row_ok);        // nothing of this warp is written
      float m = -INFINITY, l = 0.f;
      for (int j = w.j0; j < w.j1; ++j, ++it) {
        const uint32_t sb = lanes + C::COL_S + (it & 1) * kBlockKeys;
        const float* sc = s_sc + (it % C::SC_RING) * 4 * kBlockKeys + h * 64;
        if (E4) wait(sc_full + it % C::SC_RING, (it / C::SC_RING) & 1);
        wait(s_full + (it & 1), (it >> 1) & 1);
        if (idle) {
          if (lane == 0) {
            mbar_arrive_remote(mapa(smem_u32(p_ready + (it & 1)), 0));
            if (E4) mbar_arrive(sc_empty + it % C::SC_RING);
          }
          continue;
        }
        tc_fence_after();
        const int lim = last - j * kBlockKeys;                    // last visible key of the block
        const bool masked = __any_sync(0xffffffffu, lim < kBlockKeys - 1);
        unsigned long long see = ~0ull;                           // this half's visible columns
        if (masked) {
          // columns from t0 hold the sequence's last page, `shift` columns late
          const int valid = w.s.kv - j * kBlockKeys;
          int t0 = kBlockKeys, shift = 0;
          if (valid > 0 && valid < kBlockKeys) {
            t0 = (valid - 1) / ps * ps;
            shift = t0 + ps - valid;
          }
          auto below = [&](int n) {
            n -= 64 * h;
            return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
          };
          see = below(min(t0, lim + 1)) | (below(lim + shift + 1) & ~below(t0 + shift));
        }
        const float* ks = sc;
        if (E4 && masked) {
          // scaled and masked in place, the loops then multiply by ones: masks
          // in their code cost blocks without one as well
          ks = s_one;
#pragma unroll 1
          for (int c0 = 0; c0 < 64; c0 += 8) {
            float x[8];
            uint32_t u[8];
            tmem_ld8(sb + 64 * h + c0, x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              u[i] = __float_as_uint(see >> (c0 + i) & 1 ? x[i] * sc[c0 + i] : -INFINITY);
            tmem_st8(sb + 64 * h + c0, u);
          }
          tmem_st_wait();
        }
        // STEP columns at a time: all 64 stay in registers from the maximum to
        // the exponentials, or, with codes, where the widening warps' code
        // fills the instruction cache, a short loop reads them from TMEM twice
        // (8 columns: 974 us where 16 take 986 and all 64 took 1308; 2048
        // tokens over 14000, 8 heads x 128).  The keys' scales hold the softmax
        // scale as well: one product less a score.
        constexpr int STEP = E4 ? 8 : 64;
        float s[STEP];
        auto columns = [&](int c0, bool scaled) {
          if (STEP == 64) {
            tmem_ld32(sb + 64 * h, s);
            tmem_ld32(sb + 64 * h + 32, s + STEP / 2);
          } else {
            tmem_ld8(sb + 64 * h + c0, s);
          }
          tmem_ld_wait();
          if (E4 && scaled) {
#pragma unroll
            for (int i = 0; i < STEP / 4; ++i) {
              const float4 f = reinterpret_cast<const float4*>(ks + c0)[i];
              mul2(s[4 * i], s[4 * i + 1], f.x, f.y);
              mul2(s[4 * i + 2], s[4 * i + 3], f.z, f.w);
            }
          }
          if (!E4 && masked) {
            const unsigned long long bits = see >> c0;
            const uint32_t see2[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
#pragma unroll
            for (int i = 0; i < STEP; ++i) s[i] = see2[i >> 5] & (1u << (i & 31)) ? s[i] : -INFINITY;
          }
        };
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c0 = 0; c0 < 64; c0 += STEP) {
          columns(c0, true);
#pragma unroll
          for (int i = 0; i < STEP; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i]);
        }
        float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * (E4 ? 1.f : c);
        // the other half's maximum: both threads then decide alike
        mx = fmaxf(mx, exchange(mx));
        const bool grow = mx > m + kRescaleLog2 || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2(m - mx);
          if (grow) m = mx;
          l *= f;
          if (j > w.j0) {
            // one phase to wait for: P V of the block before came before this
            // S, and this block's waits for this warp
            wait(o_done, (it - 1) & 1);
            tc_fence_after();
            // a row that starts here holds zeros, or what its factor 0 must
            // not turn into NaN
#pragma unroll 1
            for (int i = 0; i < D / 64; ++i) {
              float o[32];
              uint32_t u[32];
              tmem_ld32(mine_o + 32 * i, o);
              tmem_ld_wait();
#pragma unroll
              for (int q = 0; q < 32; ++q) u[q] = __float_as_uint(f == 0.f ? 0.f : o[q] * f);
              tmem_st32(mine_o + 32 * i, u);
            }
            tmem_st_wait();
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        float l2[2] = {0.f, 0.f};
#pragma unroll 1
        for (int c0 = 0; c0 < 64; c0 += STEP) {
          if (STEP < 64) columns(c0, false);
          uint32_t pk[STEP / 2];
#pragma unroll
          for (int q = 0; q < STEP / 2; ++q) {
            float a = s[2 * q], b = s[2 * q + 1];
            if (E4) {
              const float4 f = reinterpret_cast<const float4*>(ks + c0)[q >> 1];
              if (q & 1) fma2(a, b, f.z, f.w, -base);
              else fma2(a, b, f.x, f.y, -base);
            } else {
              fma2(a, b, c, -base);
            }
            a = ex2(a);
            b = ex2(b);
            add2(l2[0], l2[1], a, b);
            if (E4) {
              const float4 f = reinterpret_cast<const float4*>(sc + kBlockKeys + c0)[q >> 1];
              if (q & 1) mul2(a, b, f.z, f.w);
              else mul2(a, b, f.x, f.y);
            }
            pk[q] = Elem<T>::from_f2(a, b);
          }
          // P of a half goes over the S columns that its own threads have read
          if (STEP == 64) tmem_st32(sb + 64 * h, pk);
          else tmem_st4(sb + 64 * h + c0 / 2, pk);
        }
        l += l2[0] + l2[1];
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_remote(mapa(smem_u32(p_ready + (it & 1)), 0));
          if (E4) mbar_arrive(sc_empty + it % C::SC_RING);
        }
      }
      if (!idle) l += exchange(l);
      // a barrier of its own: o_done may be two phases behind here
      wait(o_last, pieces & 1);
      ++pieces;
      tc_fence_after();
      const bool whole = w.j0 == 0 && w.j1 == w.nb;
      const int place = pair * 2 + (w.j0 == 0 ? 1 : 0), row = (int)rank * 128 + rr;
      if (!whole && h == 0) {
        ws.ml[((size_t)place * 256 + row) * 2] = m;
        ws.ml[((size_t)place * 256 + row) * 2 + 1] = l;
      }
      // the sum is NaN for a row of NaN scores, 0 for one of -inf alone; a row
      // that sees no key is known by its mask
      const float inv = 1.f / l;
      const bool sees = last >= 0;
      if (idle || !ok) {
      } else if (whole) {
        // four lanes swap 16-byte pieces of their four rows, so that a store
        // writes 64 neighbouring bytes of eight rows, not 16 bytes of 32
        const long long mine = (long long)(w.s.q0 + tok) * p.out_token + (long long)(w.head * p.group + hd) * p.out_head;
        T* dst[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const long long o = __shfl_sync(0xffffffffu, row_ok ? mine : -1, (lane & ~3) + k);
          dst[k] = o < 0 ? nullptr : static_cast<T*>(p.out) + o + h * (D / 2) + (lane & 3) * 8;
        }
#pragma unroll 1
        for (int i = 0; i < D / 64; ++i) {
          float o[32];
          tmem_ld32(mine_o + 32 * i, o);
          tmem_ld_wait();
          uint32_t u[4][4];                    // [piece][word]
#pragma unroll
          for (int q = 0; q < 16; ++q)
            u[q >> 2][q & 3] = sees ? Elem<T>::from_f2(o[2 * q] * inv, o[2 * q + 1] * inv) : 0u;
#pragma unroll
          for (int x = 1; x <= 2; x <<= 1) {
            const bool up = lane & x;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (!(q & x)) {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? u[q][y] : u[q | x][y], x);
                  if (up) u[q][y] = got;
                  else u[q | x][y] = got;
                }
              }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (dst[k]) *reinterpret_cast<uint4*>(dst[k] + 32 * i) = make_uint4(u[k][0], u[k][1], u[k][2], u[k][3]);
          __syncwarp();
        }
      } else {
        // [D / 4][256 rows][4]: a store of 32 rows is 512 neighbouring bytes
        float4* wo = reinterpret_cast<float4*>(ws.o) + ((size_t)place * (D / 4) + h * (D / 8)) * 256 + row;
#pragma unroll 1
        for (int i = 0; i < D / 64; ++i) {
          float o[32];
          tmem_ld32(mine_o + 32 * i, o);
          tmem_ld_wait();
          if (row_ok) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              wo[(8 * i + q) * 256] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa(smem_u32(o_free), 0));
    }
    if (rank == 0 && tid == 0) {
      // a tile that begins and does not end in this part is its last piece
      if (w.j0 == 0 && w.j1 > 0 && w.j1 < w.nb) {
        // the part that holds the tile's last block
        const long long u = (long long)part.begin + part.count + (w.nb - w.j1) - 1;
        ws.desc[2 * pair] = make_int4(w.s.q0, w.s.n, w.head, w.tile);
        ws.desc[2 * pair + 1] = make_int4(part_of(part.total, min(pairs, part.total), u), w.s.kv - w.s.n, 0, 0);
      } else {
        ws.desc[2 * pair + 1] = make_int4(-1, 0, 0, 0);
      }
    }
  } else if (E4 && warp == 11) {
    // ---- scales: lane has columns lane + 32 i of every block, in the order
    // of the loaded rows; the next block's are on their way while one is stored
    ChunkWalk walk(part, MORE);
    ChunkPiece w;
    uint32_t it = 0;
    int j = 0;
    bool more = walk.next(p, per, w);
    j = more ? w.j0 : 0;
    float k[4], v[4];
    PageWindow pages;
    auto load = [&]() {
      pages.reach(p, w.b, (j * kBlockKeys) >> p.page_shift);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int plane, row;
        pages.row(p, w, j * kBlockKeys + lane + 32 * i, plane, row);
        const bool have = plane >= 0 && row >= 0;
        const long long at_row = ((long long)plane << p.page_shift) + row;
        k[i] = have ? __ldcg(p.k_scale + at_row) : 0.f;
        v[i] = have ? __ldcg(p.v_scale + at_row) : 0.f;
      }
    };
    if (more) load();
    while (more) {
      float ck[4], cv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ck[i] = k[i];
        cv[i] = v[i];
      }
      if (++j >= w.j1) {
        more = walk.next(p, per, w);
        j = more ? w.j0 : 0;
      }
      if (more) load();
      if (!wait_warp(sc_empty + it % C::SC_RING, ((it / C::SC_RING) & 1) ^ 1, kAttnErrChunkWiden)) break;
      float* sc = s_sc + (it % C::SC_RING) * 4 * kBlockKeys + lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // v = f * 2^e; a scale without an exponent of its own stays whole
        const uint32_t b = __float_as_uint(cv[i]);
        const bool normal = (b & 0x7f800000u) != 0;
        sc[32 * i] = ck[i] * p.scale_log2;
        sc[kBlockKeys + 32 * i] = normal ? __uint_as_float((b & 0x007fffffu) | 0x3f800000u) : 1.f;
        uint32_t* e = reinterpret_cast<uint32_t*>(sc) + 2 * kBlockKeys + 32 * i;
        if (std::is_same<T, __half>::value) {
          // 2^e as two fp16 factors, each twice: fp16 codes are multiplied by
          // them (a scale without an exponent is below fp16's least)
          const int x = (int)(b >> 23 & 0xff) - 127, x1 = max(-14, min(15, x)), x2 = max(-24, min(15, x - x1));
          const uint32_t h1 = normal ? ((uint32_t)(x1 + 15) << 10) | (b >> 16 & 0x8000u) : 0u;
          const uint32_t h2 = x2 >= -14 ? (uint32_t)(x2 + 15) << 10 : 1u << (x2 + 24);
          e[0] = h1 | h1 << 16;
          e[kBlockKeys] = h2 | h2 << 16;
        } else {
          e[0] = normal ? b & 0xff800000u : b;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sc_full + it % C::SC_RING);
      ++it;
    }
  } else if (E4 && warp >= 12) {
    // ---- codes to 16 bits: raw ring -> operand ring
    const int t = tid - 384;
    ChunkTiles tl(part, MORE);
    int slot = 0, raw = 0;
    uint32_t phase = 0, raw_phase = 0, vn = 0;
    auto widen = [&](auto is_v) {
      constexpr bool v = decltype(is_v)::value;
      // ACROSS threads along a row (of half the dims, V), eight codes each.  A
      // thread's rows are a multiple of eight apart: its places in the swizzle
      // are a constant apart, which keeps the loop's code short.  The kernel is
      // bound by instruction-cache misses: this, and masks outside the softmax's
      // loops, took 2048 tokens over 14000 from 1220 to 986 us (8 heads x 128)
      // and from 731 to 642 us (2 heads x 256).
      constexpr int COLS = v ? D / 2 : D, ROWS = v ? kBlockKeys : 64, ACROSS = (COLS < 128 ? COLS : 128) / 8;
      constexpr int DOWN = 128 / ACROSS, WIDE = COLS / 8 / ACROSS;
      const int r0 = t / ACROSS, c0 = t % ACROSS;
      if (!wait_warp(raw_full + raw, raw_phase, kAttnErrChunkWiden)) return;
      if (v && !wait_warp(sc_full + vn % C::SC_RING, (vn / C::SC_RING) & 1, kAttnErrChunkWiden)) return;
      if (!wait_warp(empty + slot, phase ^ 1, kAttnErrChunkWiden)) return;
      const uint8_t* src = s_codes + (size_t)raw * C::RAW + r0 * COLS + c0 * 8;
      const uint32_t* e2 = reinterpret_cast<const uint32_t*>(s_sc) + ((vn % C::SC_RING) * 4 + 2) * kBlockKeys + r0;
      uint8_t* dst = s_ring + (size_t)slot * C::SLOT + (c0 >> 3) * (ROWS * 128) + r0 * 128 + (((c0 ^ r0) & 7) << 4);
#pragma unroll 2
      for (int i = 0; i < ROWS / DOWN * WIDE; ++i) {
        const int down = i / WIDE * DOWN, wide = i % WIDE;
        const uint2 u = *reinterpret_cast<const uint2*>(src + down * COLS + wide * 128);
        const uint32_t ea = v ? e2[down] : 0u, eb = v && std::is_same<T, __half>::value ? e2[down + kBlockKeys] : 0u;
        const uint32_t w2[2] = {u.x, u.y};
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint16_t c = (uint16_t)(w2[q >> 1] >> (16 * (q & 1)));
          o[q] = v ? widen2<T>(c, ea, eb) : widen2<T>(c);
        }
        *reinterpret_cast<uint4*>(dst + down * 128 + wide * (2 * ROWS * 128)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_remote(mapa(smem_u32(full + slot), 0));
        mbar_arrive(raw_empty + raw);
        if (v) mbar_arrive(sc_empty + vn % C::SC_RING);
      }
      if (v) ++vn;
      if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
      if (++raw == C::RAWS) { raw = 0; raw_phase ^= 1; }
    };
    while (ok && tl.next(p, per)) {
      if (tl.is_v) widen(std::true_type{});
      else widen(std::false_type{});
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // every MMA of the pair, and every arrival that it makes here, has ended
  // before TMEM or shared memory goes
  if (warp == 8 && !mbar_wait(all_done, 0, kAttnWaitBudgetNs) && lane == 0) attn_error(p.err, kAttnErrChunkMma);
  __syncwarp();
  if (p.beside) pdl_wait();
  cluster_sync_all();      // no CTA leaves while its pair may still arrive at it
  tc_fence_after();
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Tiles that the parts' cuts go through: the sum of their parts, in order.
// c0 and c1 are the first and the last of a tile's parts.  A block takes 16
// rows: a warp eight of them (a load of eight rows' 16 bytes is a whole line)
// and a quarter of the dims.
constexpr int kJoinRows = 16;
// those of a tile with rows in CTA `half` of the pair
__device__ __forceinline__ int chunk_join_groups(const AttnParams& p, const int4& de, int half) {
  const int tpc = 128 / p.group, toks = min(de.y - (de.w * 2 + half) * tpc, tpc);
  return toks > 0 ? (toks * p.group + kJoinRows - 1) / kJoinRows : 0;
}
template <typename T, int D>
__device__ __forceinline__ void chunk_join(const AttnParams& p, const ChunkWs& ws, const int4& de, int c0, int c1,
                                           int last_key, int group) {
  constexpr int N = D / 64;
  const int g0 = chunk_join_groups(p, de, 0), half = group >= g0, tpc = 128 / p.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rr = (half ? group - g0 : group) * kJoinRows + (warp & 1) * 8 + (lane & 7), row = half * 128 + rr;
  const int x = (warp >> 1) * (D / 16) + (lane >> 3);
  const int ti = rr / p.group, tok = (de.w * 2 + half) * tpc + ti;
  if (ti >= tpc || tok >= de.y) return;
  // two parts at a time (a tile seldom has more), all of their loads at once
  float m = -INFINITY, l = 0.f;
  float4 a[N];
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = c0; c <= c1; c += 2) {
    float2 ml[2];
    float4 v[2][N];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (c + k <= c1) {
        const size_t place = (size_t)(c + k) * 2 + (c + k == c0);
        ml[k] = __ldcg(reinterpret_cast<const float2*>(ws.ml) + place * 256 + row);
#pragma unroll
        for (int i = 0; i < N; ++i)
          v[k][i] = __ldcg(reinterpret_cast<const float4*>(ws.o) + (place * (D / 4) + x + 4 * i) * 256 + row);
      }
    }
    const float top = fmaxf(m, fmaxf(ml[0].x, ml[1].x)), base = top == -INFINITY ? 0.f : top;
    const float keep = ex2(m - base);
    m = top;
    l *= keep;
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = make_float4(a[i].x * keep, a[i].y * keep, a[i].z * keep, a[i].w * keep);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float f = ex2(ml[k].x - base);
      l = fmaf(ml[k].y, f, l);
      if (f == 0.f) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i].x = fmaf(v[k][i].x, f, a[i].x);
        a[i].y = fmaf(v[k][i].y, f, a[i].y);
        a[i].z = fmaf(v[k][i].z, f, a[i].z);
        a[i].w = fmaf(v[k][i].w, f, a[i].w);
      }
    }
  }
  const float inv = 1.f / l;
  const bool sees = last_key + tok >= 0;
  T* dst = static_cast<T*>(p.out) + (long long)(de.x + tok) * p.out_token +
           (long long)(de.z * p.group + rr - ti * p.group) * p.out_head + x * 4;
#pragma unroll
  for (int i = 0; i < N; ++i)
    *reinterpret_cast<uint2*>(dst + 16 * i) =
        sees ? make_uint2(Elem<T>::from_f2(a[i].x * inv, a[i].y * inv), Elem<T>::from_f2(a[i].z * inv, a[i].w * inv))
             : make_uint2(0u, 0u);
}

// What the row kernel (parts [0, rows_parts)) and the chunk kernel cut.  After
// the row kernel alone a block has one part's row, if there is one (x: part, y:
// row): the least latency.  Else every block reads the list of all parts, at
// most one a thread, and takes its share of the rows to be joined: a block for
// each 32 rows that might be cut spent more on blocks without work (24
// sequences of 3 to 7 tokens: 55.1 us in all, 51.9 with the list; 12 mixed
// ones 146 and 139; 2048 tokens 40.1 and 35.9; but one single token 9.1 and
// 10.0).
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, kJoinBlocks) attn_join_kernel(const __grid_constant__ AttnParams p, int rows_per,
                                                                    int rows_parts, int parts, const ChunkWs ws) {
  __shared__ int s_sum[kJoinThreads / 32], s_c0, s_c1, s_last, s_at;
  __shared__ int4 s_de;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  int4 de = make_int4(0, 0, 0, 0);
  int2 to = make_int2(-1, 0);    // last part, last key of the first new token
  int n = 0;
  auto read_to = [](const int4* at) {
    const int4 v = __ldcg(at);
    return make_int2(v.x, v.y);
  };
  if (gridDim.y > 1) {
    const int part = blockIdx.x, row = blockIdx.y;
    de = __ldcg(p.ws_desc + 2 * part);
    to = read_to(p.ws_desc + 2 * part + 1);
    if (to.x >= 0 && de.w * rows_per + row < de.y) rows_join<T, D>(p, rows_per, de, part, to.x, to.y, row);
    return;
  }
  const int c0 = tid < rows_parts ? tid : tid - rows_parts;
  if (tid < parts) {
    const int4* at = (tid < rows_parts ? p.ws_desc : ws.desc) + 2 * c0;
    de = __ldcg(at);
    to = read_to(at + 1);
    if (to.x >= 0)
      n = tid < rows_parts ? min(rows_per, de.y - de.w * rows_per)
                           : chunk_join_groups(p, de, 0) + chunk_join_groups(p, de, 1);
  }
  int before = n, total = 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) s_sum[warp] = before;
  __syncthreads();
  before -= n;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    if (w < warp) before += s_sum[w];
    total += s_sum[w];
  }
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    if (i >= before && i < before + n) {
      s_de = de;
      s_c0 = c0 + (tid < rows_parts ? 0 : rows_parts);
      s_c1 = to.x;
      s_last = to.y;
      s_at = i - before;
    }
    __syncthreads();
    if (s_c0 < rows_parts) rows_join<T, D>(p, rows_per, s_de, s_c0, s_c1, s_last, s_at);
    else chunk_join<T, D>(p, ws, s_de, s_c0 - rows_parts, s_c1, s_last, s_at);
    __syncthreads();
  }
}

}  // namespace d3
