// Attention of few query rows over a paged K/V cache: decode tokens, or a few
// drafted ones.
//
// The rows of one KV head (tokens x the G query heads that share it, at most
// 8 * NT of them) ride along while the head's keys and values are read once,
// so the kernel is bound by HBM: D * 2 elements per key against 4 * rows * D
// operations.  The products are mma.sync with the KEYS as the tall side,
//
//   S^T [16 keys x 8 rows]  = K [16 x D] . Q^T        (A = K,   B = Q^T)
//   O^T [16 dims x 8 rows] += V^T [16 x 16 keys] . P^T (A = V^T, B = P^T)
//
// because 8 rows fill the short side exactly, where the usual form would pad
// them to 16.  (The 128-row tcgen05 form would leave 15/16 of its rows empty;
// it takes over above 16 rows, attn_chunk.cuh.)  P^T goes from the accumulator
// layout to the operand layout with one movmatrix per 8 x 8 block.
//
// Streaming: four threads issue TMA loads (128-byte swizzle) of KEYS-key tiles of
// K and V into a ring of 32 KiB slots; each of eight (or four) warps takes 16 keys
// of every tile with a running maximum and sum of its own, so no barrier runs
// inside the stream; the warps' results are joined once a segment.
//
// Split: the tiles of all (sequence, KV head) pairs form one list that is cut
// into gridDim.x equal parts, so ragged batches load every SM alike.  A part
// holds whole pairs and at most two pieces of pairs, whose unnormalised sums
// go to the workspace (two places per CTA) and are joined by
// attn_join_kernel in the order of the parts: results do not depend on timing.
// Measured: 4 tokens over 8 heads x 100000 and more keys read 6.7 TB/s, 64
// ragged sequences of codes 4.4 (a warp's products and softmax of a tile come one
// after the other; a piece costs its start and its join); one token over a short
// context is 9 us of latency.
//
// e4m3 caches: codes are exact in fp16, so the products run in fp16 whatever
// the queries' type.  bf16 queries are scaled by a power of two per row that
// brings the largest into [2^14, 2^15), the top of fp16: their eight bits stay
// whole but for elements 2^31 times smaller than it.  A key's scale multiplies
// its scores in fp32; a value's scale, in units of a power of two not below any
// scale the warp has met, multiplies the probability before it is rounded to
// fp16.  The product is at most 1 and goes into fp16 times 2^15, so that its
// eleven bits are whole down to 2^-29 of that unit and something is left down to
// 2^-40: a row that hardly heeds a key of far larger values keeps the others'.
#pragma once

#include "kv_common.cuh"
#include "ring_drain.h"

#include <cuda.h>

#include <type_traits>

namespace d3 {

constexpr float kCodesUp = 0x1p15f;        // of probability times scale, in fp16
constexpr uint64_t kAttnWaitBudgetNs = 2000000000ull;
constexpr int kJoinThreads = 256, kJoinBlocks = 3;   // of the joining kernel: threads, blocks an SM
constexpr int kAttnErrRowsLoad = 51, kAttnErrRowsUse = 52, kAttnErrOffsets = 58;

struct AttnParams {
  const void* q;                 // [tokens][heads][D]
  long long q_token, q_head;     // strides in elements
  void* out;
  long long out_token, out_head;
  const int* table;              // [batch][table_stride] page ids
  long long table_stride;
  int table_pages;               // usable entries of a table row
  const int* kv_lens;            // [batch]
  const int* cu_q;               // [batch + 1], or NULL: one row a sequence
  int batch, tokens, heads, group, kv_heads;
  int page_size, page_shift, pages;
  const void *k_codes, *v_codes; // the cache's buffers
  const float *k_scale, *v_scale;
  float scale_log2;              // softmax scale * log2(e)
  int min_rows, max_rows;        // sequences this launch takes, by new tokens * group
  int beside;                    // the launch before is the row kernel of the same call: what that one
                                 // waited for has ended, and it itself is waited for at the end
  float* ws_o;                   // partial sums
  float* ws_ml;                  // their maxima and sums
  int4* ws_desc;                 // two of each part: (first query token, rows of the sequence, KV head, row
                                 // group), (last part or -1, last key of token 0, ...) of the pair that begins
                                 // and does not end in it
  int* err;
};

__device__ __forceinline__ void attn_error(int* err, int code) { atomicCAS(err, 0, code); }

// The rest of a wait whose first try failed, for one thread or all lanes of a
// warp: false once it has run out, with the error recorded, or *abort is set.
// Out of line: a kernel's roles run from different places of its code at once
// and its many waits in line cost it instruction-cache misses (a chunk of 2048
// over 30720: 796 us in line, 728 so, on one box; the walks out of line, with their state
// in local memory, made everything slower).
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, int* err, int code, volatile int* abort) {
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > kAttnWaitBudgetNs) {
      attn_error(err, code);
      *abort = 1;
      return false;
    }
  }
}

struct AttnSeq {
  int q0, n, kv, rows;           // first query token, new tokens, keys, rows of a KV head
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& p, int b) {
  AttnSeq s;
  if (p.cu_q) {
    s.q0 = __ldcg(p.cu_q + b);
    s.n = __ldcg(p.cu_q + b + 1) - s.q0;
  } else {
    s.q0 = b;
    s.n = 1;
  }
  // offsets outside the query tensor (a broken cu_q) are cut to it
  if (s.q0 < 0 || s.q0 > p.tokens) s.n = 0;
  else s.n = max(0, min(s.n, p.tokens - s.q0));
  s.kv = max(0, min(__ldcg(p.kv_lens + b), p.table_pages * p.page_size));
  s.rows = s.n * p.group;
  return s;
}

template <typename T, int D, bool E4, int NT>
struct RowsCfg {
  static constexpr int ES = E4 ? 1 : 2;                     // bytes of a cached element
  static constexpr int WARPS = (D == 256 && (!E4 || NT == 2)) ? 4 : 8;   // consumer warps: registers for D = 256
  static constexpr int KEYS = 16 * WARPS;
  static constexpr int LOADERS = 4;                         // loading warps, one thread each
  static constexpr int THREADS = 32 * (WARPS + LOADERS);
  static constexpr int COLS = D * ES / 128;                 // 128-byte columns of a row
  static constexpr int ROWS = 8 * NT;
  static constexpr int SLOT = KEYS * D * ES;                // 32 KiB, 16 KiB for D = 128 codes
  static constexpr int QFRAG = NT * D * 16;
  // warps' results are joined DC dims at a time through 32 KiB
  static constexpr int DC = (32 * 1024) / (WARPS * ROWS * 4) < D ? (32 * 1024) / (WARPS * ROWS * 4) : D;
  static constexpr int JOIN_PITCH = DC + 4;
  static constexpr int JOIN = WARPS * ROWS * JOIN_PITCH * 4;
  static constexpr int SLOTS = (222 * 1024 - QFRAG - JOIN) / SLOT < 10
                                   ? (222 * 1024 - QFRAG - JOIN) / SLOT : 10;
  static constexpr int ML = WARPS * ROWS * 2 * 4;
  static constexpr size_t SMEM = 1024 + (size_t)SLOTS * SLOT + QFRAG + JOIN + ML + 4 * ROWS + 256;
  static_assert(SLOTS >= 4, "the ring needs two tiles in flight");
};

// A part of the list: where it begins and how long it is.  Every pair stands
// in the list with its tiles and kPieceUnits more in front of them, about what
// a piece costs besides (queries in, results joined and out), so that parts of
// many short pairs are as long as those of one.
constexpr int kPieceUnits = 1;
struct RowsWork {
  int total, begin, count;
  int b, off;                    // sequence of `begin`, and its place inside it
  AttnSeq s;
};

__device__ __forceinline__ int rows_tiles(int kv, int keys) { return max(1, (kv + keys - 1) / keys); }

// Lengths of the list add up to kListMost at most.  The host has checked that
// sequences which share no row stay below it; offsets that go back and forth
// can give every sequence all of the rows.  A list that reaches it has no parts:
// the kernel records an error and writes nothing.
constexpr int kListMost = 0x7fffffff;
__device__ __forceinline__ int list_add(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kListMost); }
__device__ __forceinline__ int list_total(const AttnParams& p, int total) {
  if (total < kListMost) return total;
  if (threadIdx.x == 0) attn_error(p.err, kAttnErrOffsets);
  return 0;
}
// units of sequence b over all of its KV heads and row groups
__device__ __forceinline__ int rows_units(const AttnParams& p, int b, int keys, int rows_per) {
  const AttnSeq s = attn_seq(p, b);
  if (s.rows == 0 || s.rows < p.min_rows || s.rows > p.max_rows) return 0;
  return (rows_tiles(s.kv, keys) + kPieceUnits) * p.kv_heads * ((s.rows + rows_per - 1) / rows_per);
}
// where part c of g equal ones begins
__device__ __forceinline__ int part_begin(int total, int g, int c) {
  const int q = total / g;
  return q * c + (total - q * g) * c / g;
}
// the part that holds unit u
__device__ __forceinline__ int part_of(int total, int g, long long u) { return (int)(((u + 1) * g - 1) / total); }

// All threads of the CTA: part `part` of `parts`.  s_scan: 32 ints of shared memory.
__device__ RowsWork rows_plan(const AttnParams& p, int keys, int rows_per, int part, int parts, int* s_scan, RowsWork* s_work) {
  const int n = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.batch + n - 1) / n;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  int sum = 0;
  for (int b = b0; b < b1; ++b) sum = list_add(sum, rows_units(p, b, keys, rows_per));
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc = list_add(inc, v);
  }
  if (lane == 31) s_scan[warp] = inc;
  __syncthreads();
  int before = inc - sum, total = 0;
  for (int w = 0; w < n / 32; ++w) {
    if (w < warp) before = list_add(before, s_scan[w]);
    total = list_add(total, s_scan[w]);
  }
  total = list_total(p, total);
  RowsWork r{total, 0, 0, 0, 0, {0, 0, 0, 0}};
  // no part is empty: a pair's parts are neighbours in the workspace
  const int g = min(parts, total);
  if (part < g) {
    r.begin = part_begin(total, g, part);
    r.count = part_begin(total, g, part + 1) - r.begin;
  }
  if (r.count > 0 && before <= r.begin && r.begin < before + sum) {
    int at = before;
    for (int b = b0; b < b1; ++b) {
      const int u = rows_units(p, b, keys, rows_per);
      if (r.begin < at + u) {
        r.b = b;
        r.off = r.begin - at;
        r.s = attn_seq(p, b);
        *s_work = r;
        break;
      }
      at += u;
    }
  }
  if (r.count == 0 && tid == 0) *s_work = r;
  __syncthreads();
  return *s_work;
}

// One piece of a (sequence, KV head, row group): tiles [t0, t1) of nt.
struct RowsPiece {
  AttnSeq s;
  int b, head, rg, t0, t1, nt;
};
// Walks a part of the list piece by piece.
struct RowsWalk {
  int b, left, off;
  int known;                     // the sequence that s holds
  AttnSeq s;
  __device__ __forceinline__ explicit RowsWalk(const RowsWork& r) : b(r.b), left(r.count), off(r.off), known(r.b), s(r.s) {}
  __device__ __forceinline__ bool next(const AttnParams& p, int keys, int rows_per, RowsPiece& w) {
    while (left > 0 && b < p.batch) {
      if (known != b) {
        s = attn_seq(p, b);
        known = b;
      }
      if (s.rows > 0 && s.rows >= p.min_rows && s.rows <= p.max_rows) {
        const int nt = rows_tiles(s.kv, keys), len = nt + kPieceUnits;
        const int groups = (s.rows + rows_per - 1) / rows_per;
        if (off < len * p.kv_heads * groups) {
          const int hg = off / len, pos = off - hg * len, take = min(left, len - pos);
          left -= take;
          off += take;
          w.s = s;
          w.b = b;
          w.nt = nt;
          w.head = hg / groups;
          w.rg = hg - w.head * groups;
          w.t0 = max(0, pos - kPieceUnits);
          w.t1 = max(0, pos + take - kPieceUnits);
          if (w.t1 > w.t0) return true;
          continue;              // nothing but the units in front
        }
      }
      ++b;
      off = 0;
    }
    return false;
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                      uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1,
                                                     uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16-byte piece (of 8 a 128-byte column) of row `key` of a swizzled box whose
// columns are `col` bytes apart
__device__ __forceinline__ uint32_t tile_piece(uint32_t base, uint32_t col, int key, int piece) {
  return base + (uint32_t)(piece >> 3) * col + key * 128 + (((piece ^ key) & 7) << 4);
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z, int u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x),
      "r"(y), "r"(z), "r"(u)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T, int D, bool E4, int NT>
__global__ void __launch_bounds__(RowsCfg<T, D, E4, NT>::THREADS, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ AttnParams p) {
  using C = RowsCfg<T, D, E4, NT>;
  using M = typename std::conditional<E4, __half, T>::type;   // operand type of the products
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_scan[32];
  __shared__ RowsWork s_work;
  __shared__ volatile int s_abort;
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* s_slots = smem;
  uint2* s_q = reinterpret_cast<uint2*>(smem + (size_t)C::SLOTS * C::SLOT);
  float* s_join = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + C::QFRAG);
  float* s_ml = s_join + C::JOIN / 4;                          // [WARPS][ROWS][2]
  float* s_qs = s_ml + C::ML / 4;                              // [ROWS] scale of a row's scores
  uint64_t* full = reinterpret_cast<uint64_t*>(s_qs + C::ROWS + (C::ROWS & 1));
  uint64_t* empty = full + C::SLOTS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(full + i, C::LOADERS);
      mbar_init(empty + i, C::WARPS);
    }
    fence_barrier_init();
    s_abort = 0;
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // in this order: the chunk kernel behind may then run beside this one
  pdl_wait();
  pdl_trigger();
  const RowsWork work = rows_plan(p, C::KEYS, C::ROWS, blockIdx.x, gridDim.x, s_scan, &s_work);
  if (work.count == 0) {
    if (tid == 0) p.ws_desc[2 * blockIdx.x + 1] = make_int4(-1, 0, 0, 0);
    return;
  }
  RowsWalk walk(work);
  RowsPiece w{};
  const int box = min(p.page_size, C::KEYS), boxes = C::KEYS / box;     // rows of a TMA box, boxes of a tile
  if (warp >= C::WARPS) {
    // ---- loading threads: K tile, V tile, K tile, ...  A box is a page's
    // rows with all of their columns, so a tile is [boxes][columns][box rows]
    // [128 bytes]; thread i takes boxes i, i + 4.  (A TMA instruction holds
    // its thread for some 300 cycles whatever its size, so small pages need
    // several threads.)  The page ids of the next tile are on their way while
    // this one's boxes go out.
    if (lane == 0) {
      const int who = warp - C::WARPS;
      constexpr int MINE = 8 / C::LOADERS;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      int t = 0, ids[MINE];
      auto fetch = [&]() {
        const int* row = p.table + (long long)w.b * p.table_stride;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
          const int key = t * C::KEYS + (who + i * C::LOADERS) * box;
          ids[i] = who + i * C::LOADERS < boxes && key < w.s.kv ? __ldcg(row + (key >> p.page_shift)) : -1;
        }
      };
      bool more = walk.next(p, C::KEYS, C::ROWS, w);
      if (more) {
        t = w.t0;
        fetch();
      }
      while (more && ok) {
        const int key0 = t * C::KEYS, head = w.head;
        // keys of this tile in whole boxes: what lies behind is never loaded
        const int need = min(boxes, (max(0, w.s.kv - key0) + box - 1) / box);
        int plane[MINE];
#pragma unroll
        for (int i = 0; i < MINE; ++i)
          plane[i] = ids[i] >= 0 && ids[i] < p.pages ? ids[i] * p.kv_heads + head : -1;
        const int in_page = key0 & (p.page_size - 1);    // of the first box, where a page is larger than a tile
        if (++t >= w.t1) {
          more = walk.next(p, C::KEYS, C::ROWS, w);
          if (more) t = w.t0;
        }
        if (more) fetch();
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (!mbar_try_wait(empty + slot, phase ^ 1) &&
              !wait_on(smem_u32(empty + slot), phase ^ 1, p.err, kAttnErrRowsLoad, &s_abort)) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(s_slots + (size_t)slot * C::SLOT);
          // every thread arrives, boxes or not: a thread that has none in some
          // tiles would else be overtaken by two turns of the ring, and wait
          // for a phase that has come and gone
          if (who == 0) mbar_arrive_expect_tx(full + slot, need * box * D * C::ES);
          else mbar_arrive(full + slot);
          // a page id outside the cache is loaded from outside the map: zeros
#pragma unroll
          for (int i = 0; i < MINE; ++i)
            if (who + i * C::LOADERS < need)
              tma_load_4d(dst + (who + i * C::LOADERS) * box * (D * C::ES), kv ? &tm_v : &tm_k, smem_u32(full + slot),
                          0, in_page, 0, plane[i]);
          if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
        }
      }
      // what is still in flight has landed before the CTA's memory goes
      if (!ok)
        drain_ring(C::SLOTS, slot, phase, kAttnWaitBudgetNs,
                   [&](int i, uint32_t par) { return mbar_try_wait(full + i, par); },
                   [] { return globaltimer_ns(); });
    }
    return;
  }

  // ---- the other warps: 16 keys of every tile
  const int g = lane >> 2, t4 = lane & 3;
  // this warp's 16 keys of a tile lie in one box
  const uint32_t col = box * 128, mine = warp * 16 / box * (box * D * C::ES) + warp * 16 % box * 128;
  int slot = 0;
  uint32_t phase = 0;
  bool ok = true;
  auto bar = [&]() { asm volatile("bar.sync 1, %0;" ::"r"(C::WARPS * 32) : "memory"); };
  auto take = [&]() {
    if (ok && !__all_sync(0xffffffffu, mbar_try_wait(full + slot, phase)))
      ok = __all_sync(0xffffffffu, wait_on(smem_u32(full + slot), phase, p.err, kAttnErrRowsUse, &s_abort));
  };
  auto give = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + slot);
    if (++slot == C::SLOTS) { slot = 0; phase ^= 1; }
  };
  // a piece's queries are fetched while the one before runs: this warp's rows,
  // 16 bytes a lane
  constexpr int QROWS = (C::ROWS + C::WARPS - 1) / C::WARPS;
  uint4 q_next[QROWS];
  auto fetch_q = [&](const RowsPiece& x) {
#pragma unroll
    for (int k = 0; k < QROWS; ++k) {
      const int r = warp + k * C::WARPS, gr = x.rg * C::ROWS + r;
      q_next[k] = make_uint4(0, 0, 0, 0);
      if (r < C::ROWS && gr < x.s.rows && lane < D / 8)
        q_next[k] = __ldcg(reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) + (long long)(x.s.q0 + gr / p.group) * p.q_token +
            (long long)(x.head * p.group + gr % p.group) * p.q_head + lane * 8));
    }
  };
  // codes: the scales of keys g and g + 8 of this warp's 16, a tile ahead, and
  // the page id they need two ahead (a piece's first ones while the piece
  // before runs)
  float ks_n[2] = {0.f, 0.f}, vs_n[2] = {0.f, 0.f};
  int id_n = -1, id_first = -1;
  auto fetch_id = [&](const RowsPiece& x, int t) {
    const int key = t * C::KEYS + warp * 16;
    return E4 && t < x.t1 && key < x.s.kv
               ? __ldcg(p.table + (long long)x.b * p.table_stride + (key >> p.page_shift)) : -1;
  };
  auto fetch_scales = [&](const RowsPiece& x, int t, int id) {
    if (!E4) return;
    const bool in = id >= 0 && id < p.pages;
    const long long row = ((long long)(in ? id * p.kv_heads + x.head : 0) << p.page_shift) +
                          ((t * C::KEYS + warp * 16) & (p.page_size - 1)) + g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ks_n[i] = in ? __ldcg(p.k_scale + row + 8 * i) : 0.f;
      vs_n[i] = in ? __ldcg(p.v_scale + row + 8 * i) : 0.f;
    }
  };
  RowsPiece ahead{};
  bool more = walk.next(p, C::KEYS, C::ROWS, ahead);
  if (more) {
    fetch_q(ahead);
    id_first = fetch_id(ahead, ahead.t0);
  }
  while (more) {
    w = ahead;
    id_n = fetch_id(w, w.t0 + 1);
    fetch_scales(w, w.t0, id_first);
    const int row0 = w.rg * C::ROWS, rows = min(C::ROWS, w.s.rows - row0);
    // queries in operand order: s_q[nt][kk][lane] holds the two registers of
    // B for k-step kk.  Codes come out of ldmatrix four dims to a lane, so
    // there the lane's k positions stand for dims 4t .. 4t + 3.
    bar();   // the piece before has read s_q and s_join
#pragma unroll
    for (int k = 0; k < QROWS; ++k) {
      const int r = warp + k * C::WARPS;
      if (r >= C::ROWS) break;
      const uint4 u = q_next[k];
      float x[8];
      unpack8<T>(u, x);
      float mul = 1.f, back = 1.f, amax = 0.f;
      if (E4 && std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // amax in [2^(e-1), 2^e) goes to [2^14, 2^15); the factor and its inverse
        // stay inside fp32's normal range
        int e = 0;
        if (amax > 0.f && amax < INFINITY) frexpf(amax, &e);
        e = max(-126, e - 15);
        mul = ldexpf(1.f, -e);
        back = ldexpf(1.f, e);
      }
      if (lane == 0) s_qs[r] = p.scale_log2 * back;
      if (lane < D / 8) {
        const uint4 o = make_uint4(Elem<M>::from_f2(x[0] * mul, x[1] * mul), Elem<M>::from_f2(x[2] * mul, x[3] * mul),
                                   Elem<M>::from_f2(x[4] * mul, x[5] * mul), Elem<M>::from_f2(x[6] * mul, x[7] * mul));
        const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
        uint32_t* fr = reinterpret_cast<uint32_t*>(s_q + (r / 8) * (D / 16) * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = lane * 8 + 2 * i, kk = d >> 4, in = (d & 15) >> 1;    // pair 0..7 of the k-step
          const int tt = E4 ? in >> 1 : in & 3, half = E4 ? in & 1 : in >> 2;
          fr[(kk * 32 + (r & 7) * 4 + tt) * 2 + half] = ow[i];
        }
      }
    }
    bar();
    more = walk.next(p, C::KEYS, C::ROWS, ahead);
    if (more) {
      fetch_q(ahead);
      id_first = fetch_id(ahead, ahead.t0);
    }
    // queries' operand, from shared memory each time where registers are short
    constexpr bool QREG = NT == 1 && !(E4 && D == 256);
    uint2 qr[QREG ? D / 16 : 1];
    if (QREG) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) qr[QREG ? i : 0] = s_q[i * 32 + lane];
    }
    auto qop = [&](int n, int kk) { return QREG ? qr[QREG ? kk : 0] : s_q[(n * (D / 16) + kk) * 32 + lane]; };
    float vref = 0.f;    // codes: the sums are in units of this power of two
    float o[NT][D / 16][4];
    float mx[NT][2], sum[NT][2], cs[NT][2];
    int last[NT][2];     // last key a row sees
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = n * 8 + 2 * t4 + j;
        mx[n][j] = -INFINITY;
        sum[n][j] = 0.f;
        cs[n][j] = s_qs[r];
        last[n][j] = r < rows ? w.s.kv - w.s.n + (row0 + r) / p.group : -1;
      }
    }
    const int lk = lane & 7, lm = lane >> 3;     // ldmatrix: row and matrix of this lane
    for (int t = w.t0; t < w.t1; ++t) {
      const int key0 = t * C::KEYS + warp * 16;  // this warp's keys
      const float ks0 = E4 ? ks_n[0] : 1.f, ks1 = E4 ? ks_n[1] : 1.f;
      float u0 = E4 ? vs_n[0] : 1.f, u1 = E4 ? vs_n[1] : 1.f;
      fetch_scales(w, t + 1, id_n);
      id_n = fetch_id(w, t + 2);
      take();
      const uint32_t kb = smem_u32(s_slots + (size_t)slot * C::SLOT) + mine;
      float s[NT][4];
      if (ok && key0 < w.s.kv) {
        float s2[NT][2][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) s2[n][c][j] = 0.f;
        if (E4) {
#pragma unroll
          for (int kk = 0; kk < D / 16; kk += 2) {
            uint32_t r[4];
            ldsm4(tile_piece(kb, col, (lm & 1) * 8 + lk, kk + (lm >> 1)), r);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t a0 = e4m3x2_to_h2((uint16_t)r[2 * c]), a2 = e4m3x2_to_h2((uint16_t)(r[2 * c] >> 16));
              const uint32_t a1 = e4m3x2_to_h2((uint16_t)r[2 * c + 1]), a3 = e4m3x2_to_h2((uint16_t)(r[2 * c + 1] >> 16));
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint2 b = qop(n, kk + c);
                mma16<M>(s2[n][c], a0, a1, a2, a3, b.x, b.y);
              }
            }
          }
        } else {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t r[4];
            ldsm4(tile_piece(kb, col, (lm & 1) * 8 + lk, 2 * kk + (lm >> 1)), r);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 b = qop(n, kk);
              mma16<M>(s2[n][kk & 1], r[0], r[1], r[2], r[3], b.x, b.y);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] = s2[n][0][j] + s2[n][1][j];
      }
      give();
      take();
      if (ok && key0 < w.s.kv) {
        const uint32_t vb = smem_u32(s_slots + (size_t)slot * C::SLOT) + mine;
        if (E4) {
          // values' scales in units of vref, a power of two not below any yet
          // (a caller's own scales may be negative)
          u0 = key0 + g < w.s.kv ? u0 : 0.f;
          u1 = key0 + g + 8 < w.s.kv ? u1 : 0.f;
          float vmax = fmaxf(fabsf(u0), fabsf(u1));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, x));
          if (vmax > vref) {
            const float up = __uint_as_float((__float_as_uint(vmax) + 0x7fffffu) & 0xff800000u);
            const float f = vref / up;
            vref = up;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][i][j] *= f;
          }
          // 1 / vref, a power of two as well, by its exponent
          const float inv = vref > 0.f ? __uint_as_float(0x7f000000u - __float_as_uint(vref)) : 0.f;
          u0 = u0 * inv * kCodesUp;
          u1 = u1 * inv * kCodesUp;
        }
        uint32_t pb[NT][2];
        float pr[NT][4], keep[NT][2], top[NT][2];
        bool same = true;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            pr[n][j] = key0 + g <= last[n][j] ? s[n][j] * (cs[n][j] * ks0) : -INFINITY;
            pr[n][2 + j] = key0 + g + 8 <= last[n][j] ? s[n][2 + j] * (cs[n][j] * ks1) : -INFINITY;
            top[n][j] = fmaxf(pr[n][j], pr[n][2 + j]);
          }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) top[n][j] = fmaxf(top[n][j], __shfl_xor_sync(0xffffffffu, top[n][j], x));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float m = fmaxf(top[n][j], mx[n][j]);
            const float base = m == -INFINITY ? 0.f : m;
            keep[n][j] = ex2(mx[n][j] - base);
            mx[n][j] = m;
            const float pa = ex2(pr[n][j] - base), pc = ex2(pr[n][2 + j] - base);
            sum[n][j] = fmaf(sum[n][j], keep[n][j], pa + pc);
            pr[n][j] = pa * u0;
            pr[n][2 + j] = pc * u1;
            same = same && keep[n][j] == 1.f;
          }
          pb[n][0] = movm(Elem<M>::from_f2(pr[n][0], pr[n][1]));
          pb[n][1] = movm(Elem<M>::from_f2(pr[n][2], pr[n][3]));
        }
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[n][i][j] *= keep[n][j & 1];
        }
        if (key0 + 16 > w.s.kv) {
          // values of keys behind the sequence's end are whatever the page
          // held, and 0 * NaN is no zero: this warp's rows are its own to clear
          for (int r = w.s.kv - key0; r < 16; ++r)
            for (int x = lane; x < D * C::ES / 16; x += 32)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile_piece(vb, col, r, x)), "r"(0) : "memory");
          // the next load of this slot writes the same bytes through the async
          // proxy, which the arrival that frees the slot does not order alone
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (E4) {
          // one 8 x 8 block of code pairs holds 16 dims: dim 2g in the even
          // bytes, 2g + 1 in the odd ones
#pragma unroll
          for (int i = 0; i < D / 16; i += 2) {
            uint32_t r[4];
            ldsm4t(tile_piece(vb, col, (lm & 1) * 8 + lk, i + (lm >> 1)), r);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t x = __byte_perm(r[2 * c], 0, 0x3120), y = __byte_perm(r[2 * c + 1], 0, 0x3120);
              const uint32_t a0 = e4m3x2_to_h2((uint16_t)x), a1 = e4m3x2_to_h2((uint16_t)(x >> 16));
              const uint32_t a2 = e4m3x2_to_h2((uint16_t)y), a3 = e4m3x2_to_h2((uint16_t)(y >> 16));
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16<M>(o[n][i + c], a0, a1, a2, a3, pb[n][0], pb[n][1]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t r[4];
            ldsm4t(tile_piece(vb, col, (lm >> 1) * 8 + lk, 2 * i + (lm & 1)), r);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16<M>(o[n][i], r[0], r[1], r[2], r[3], pb[n][0], pb[n][1]);
          }
        }
      }
      give();
    }
    // ---- join the warps: out, or this CTA's place in the workspace
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v = sum[n][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        if (g == 0) {
          float* ml = s_ml + (warp * C::ROWS + n * 8 + 2 * t4 + j) * 2;
          ml[0] = mx[n][j];
          ml[1] = v;
        }
      }
    bar();
    const bool whole = w.t0 == 0 && w.t1 == w.nt;
    const int place = blockIdx.x * 2 + (w.t0 == 0 ? 1 : 0);
    float* wo = p.ws_o + (size_t)place * C::ROWS * D;
    float f[NT][2];    // this warp's factor of its rows
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = n * 8 + 2 * t4 + j;
        float m = -INFINITY;
        for (int x = 0; x < C::WARPS; ++x) m = fmaxf(m, s_ml[(x * C::ROWS + r) * 2]);
        // a maximum leaves NaN out, a sum does not: a row of NaN scores has the
        // maximum -inf and the sum NaN, and its quotient is NaN, as is that of
        // a row whose scores are all -inf.  A row that sees no key is known by
        // its mask alone.
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        for (int x = 0; x < C::WARPS; ++x)
          l += s_ml[(x * C::ROWS + r) * 2 + 1] * ex2(s_ml[(x * C::ROWS + r) * 2] - base);
        f[n][j] = ex2(mx[n][j] - base);
        if (E4) f[n][j] *= vref * (1.f / kCodesUp);
        if (whole) f[n][j] = last[n][j] >= 0 ? f[n][j] / l : 0.f;
        else if (warp == 0 && g == 0) {
          p.ws_ml[(place * C::ROWS + r) * 2] = m;
          p.ws_ml[(place * C::ROWS + r) * 2 + 1] = l;
        }
      }
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += C::DC) {
      if (d0) bar();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < C::DC / 16; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // code blocks: dims 2g and 2g + 1 are rows g and g + 8
            const int d = i * 16 + (E4 ? 2 * g + (j >> 1) : g + (j >> 1) * 8);
            const int r = n * 8 + 2 * t4 + (j & 1);
            const float v = o[n][d0 / 16 + i][j];
            s_join[(warp * C::ROWS + r) * C::JOIN_PITCH + d] = f[n][j & 1] == 0.f ? 0.f : v * f[n][j & 1];
          }
      bar();
      for (int i = tid; i < rows * (C::DC / 4); i += C::WARPS * 32) {
        const int r = i / (C::DC / 4), d = (i - r * (C::DC / 4)) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < C::WARPS; ++x) {
          const float4 v = *reinterpret_cast<const float4*>(s_join + (x * C::ROWS + r) * C::JOIN_PITCH + d);
          a.x += v.x;
          a.y += v.y;
          a.z += v.z;
          a.w += v.w;
        }
        if (whole) {
          const int gr = row0 + r;
          T* dst = static_cast<T*>(p.out) + (long long)(w.s.q0 + gr / p.group) * p.out_token +
                   (long long)(w.head * p.group + gr % p.group) * p.out_head + d0 + d;
          *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<T>::from_f2(a.x, a.y), Elem<T>::from_f2(a.z, a.w));
        } else {
          *reinterpret_cast<float4*>(wo + (size_t)r * D + d0 + d) = a;
        }
      }
    }
  }
  if (tid == 0) {
    // a pair that begins and does not end in this part is its last piece
    if (w.t0 == 0 && w.t1 > 0 && w.t1 < w.nt) {
      // the part that holds the pair's last tile
      const long long u = (long long)work.begin + work.count + (w.nt - w.t1) - 1;
      p.ws_desc[2 * blockIdx.x] = make_int4(w.s.q0, w.s.rows, w.head, w.rg);
      p.ws_desc[2 * blockIdx.x + 1] =
          make_int4(part_of(work.total, min((int)gridDim.x, work.total), u), w.s.kv - w.s.n, 0, 0);
    } else {
      p.ws_desc[2 * blockIdx.x + 1] = make_int4(-1, 0, 0, 0);
    }
  }
}

// Pairs that the parts' cuts go through: the sum of their parts, in the parts'
// order.  c0 and c1 are the first and the last of its parts, last_key that of
// the sequence's first new token, r the row; the threads take turns of D/4 over
// the parts and add up through shared memory.  A part's sum counts even if its
// factor is 0: it may be NaN.  The workspace is read through L2: launched early, this kernel
// shares SMs with the join of the call before, whose lines of the same memory
// may still be in L1.
template <typename T, int D>
__device__ __forceinline__ void rows_join(const AttnParams& p, int rows_per, const int4& de, int c0, int c1, int last_key,
                                          int r) {
  constexpr int GROUPS = kJoinThreads / (D / 4);
  __shared__ float4 s_a[GROUPS][D / 4];
  __shared__ float2 s_ml[GROUPS];
  const int gr = de.w * rows_per + r;
  const int g = threadIdx.x / (D / 4), d4 = threadIdx.x % (D / 4);
  // a group's parts four at a time, all of their loads at once
  float m = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = c0 + g; c <= c1; c += 4 * GROUPS) {
    float2 ml[4];
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ck = c + k * GROUPS;
      ml[k] = make_float2(-INFINITY, 0.f);
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (ck <= c1) {
        const size_t at = ((size_t)ck * 2 + (ck == c0)) * rows_per + r;
        ml[k] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + at * 2));
        v[k] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D) + d4);
      }
    }
    const float top = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x));
    const float base = top == -INFINITY ? 0.f : top, keep = ex2(m - base);
    m = top;
    l *= keep;
    a = make_float4(a.x * keep, a.y * keep, a.z * keep, a.w * keep);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = ex2(ml[k].x - base);
      l = fmaf(ml[k].y, f, l);
      if (f == 0.f) continue;
      a.x = fmaf(v[k].x, f, a.x);
      a.y = fmaf(v[k].y, f, a.y);
      a.z = fmaf(v[k].z, f, a.z);
      a.w = fmaf(v[k].w, f, a.w);
    }
  }
  s_a[g][d4] = a;
  if (d4 == 0) s_ml[g] = make_float2(m, l);
  __syncthreads();
  if (g) return;
  float top = -INFINITY;
#pragma unroll
  for (int x = 0; x < GROUPS; ++x) top = fmaxf(top, s_ml[x].x);
  const float base = top == -INFINITY ? 0.f : top;
  l = 0.f;
  a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int x = 0; x < GROUPS; ++x) {
    const float f = ex2(s_ml[x].x - base);
    l = fmaf(s_ml[x].y, f, l);
    if (f == 0.f) continue;
    const float4 v = s_a[x][d4];
    a.x = fmaf(v.x, f, a.x);
    a.y = fmaf(v.y, f, a.y);
    a.z = fmaf(v.z, f, a.z);
    a.w = fmaf(v.w, f, a.w);
  }
  const float inv = 1.f / l;
  T* dst = static_cast<T*>(p.out) + (long long)(de.x + gr / p.group) * p.out_token +
           (long long)(de.z * p.group + gr % p.group) * p.out_head + d4 * 4;
  const bool sees = last_key + gr / p.group >= 0;
  *reinterpret_cast<uint2*>(dst) =
      sees ? make_uint2(Elem<T>::from_f2(a.x * inv, a.y * inv), Elem<T>::from_f2(a.z * inv, a.w * inv))
           : make_uint2(0u, 0u);
}

}  // namespace d3
