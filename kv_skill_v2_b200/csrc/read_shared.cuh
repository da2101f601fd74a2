// Shared read: the routed two-level read (xenc/injector.py:239-265) with every page fetched once for ALL query rows
// that read it, whichever Libraries they belong to: forked Libraries whose tables name the same pages, many requests
// on one document, prompts with top-k routing.
//
//   r[t] = sum_j wk[t, j] * softmax_n(read_temp * q_t . K_p[n]) @ V_p,   p = page_of[lib(t), idx[t, j]], n < n_valid
//
// The (row, routed chunk) pairs are grouped by page (count, scan, scatter); a tile is one page with up to MT of its
// pairs, a unit one tile with up to 512 of the page's slots. A cluster of 4 CTAs (8 for d_s > 2048) computes a unit on
// the 5th generation tensor cores, both products with the page as the 128-row operand and the pairs as its N:
//   scores  CTA j: S^T[its slots, pairs] = K . Q^T over all of d_s (TMA tiles, f32 in TMEM);
//   softmax the pairs' maxima exchanged through distributed shared memory, P = 2^(t - max) in 16 bits, CTA j's block of
//           P sent to every CTA of the cluster (bulk copies between their shared memories, counted on an mbarrier);
//   read    CTA j: O^T[its columns of d_s, pairs] = V^T . P^T (V as an MN-major operand), scaled by 1 / sum, stored per
//           pair: a warp's lanes are consecutive columns, so the stores are whole lines.
// The scores and the read walk the page differently (all columns of some slots, all slots of some columns), so the page
// passes through shared memory twice, but its second pass comes from L2: a cluster holds one or two pages at a time.
// The roles run one unit apart: the scores of the next unit are computed while this one's softmax and exchange run (with
// TERMS = 2 a quarter of them: the RS_ACC accumulators are drained by the softmax warps), and the epilogue stores one
// unit while the next one's P is made.
// A unit of few pairs (16 / TERMS) takes its read product on the softmax warps instead, with mma.sync: one 16-row tile
// holds all of its pairs, hi and lo together.
// shared_combine adds a row's pairs in the order of its routing: results do not depend on how pairs were grouped.
//
// Measured (f16 slots, d_s 2048, pages of 512): 64 rows of top-4 routing on 64 pages 69 us a call, the read 54 us (2.5 TB/s
// of pages); 32 forks with 48 common and 16 own pages each, dense, 424 and 364 us (3.2 TB/s); 4096 rows of top-4 routing
// to bf16 283 and 205-213 us (0.32 PFLOP/s), 22 us the split and 40 us the combine. Beside read_decode, which reads a page
// again for every pair: 79 against 114 us at 4 readers a page (64 rows), 81 against 364 at 16, 477 against 5560 at 256
// (float32 results), but 71 against 44 at 1.6 and 127 against 73 where no page is shared: it pays from about 3 readers.
//
// What bounds it, by cycle counts of the roles: a unit takes 37k cycles in both regimes. Few pairs: the scores of the next
// unit (18-20k, of them 2-5k waits for accumulators and 3-5k for stages) and the read of few pairs (18k) follow one
// another, as the same warps serve both. Many pairs: the next scores (15-17k, half of it waits for stages) and the read
// (21k, 1k of waits) follow one another on the MMA thread. The read's 128 products leave it at 158 cycles each, as its
// loops have no constant length; the product itself (M 128, N 64, K 16, V MN-major) takes 73 to 84 cycles alone, the
// scores' (both operands K-major) 48. With loops of constant length the read took 13.7k cycles.
//
// Why the page is the 128-row operand: with the pairs as the 128 rows (of which a tile fills 64) the read cost 290 cycles
// per 16 slots x 256 columns (M = 128, N = 256, MN-major B), this way two products.
//
// Precision. The operands are 16-bit. TERMS = 2 (float32 outputs, bf16 slots): q and P enter as hi + lo pairs, two of the MMA's
// N columns per pair, which keeps 22 bits with f16 slots and 16 with bf16; the halves are added in float32.
// bf16 slots take it for 16-bit outputs too: one rounding of q and P to 8 bits added half of the result's own rounding.
// TERMS = 1 (16-bit outputs of f16 slots): one rounding of q and of P, to 11 bits. q is scaled by a power of
// two per row and P by 2^14, so f16's range is no limit.
//
// The tensor core's accumulator drops bits below its running value at every 16-term step, always towards zero; over
// d_s = 2048 that is 128 steps, 1.2e-5 of a score near 1, which read_temp multiplies. With TERMS = 2 the scores are
// therefore accumulated 128 columns of d_s at a time into a ring of TMEM buffers and added up in float32 registers.
//
// Slots at or past n_valid never reach a result: their scores are masked, P is 0 there, and the rows of V behind the
// tile's last valid slot are zeroed in shared memory (0 * NaN would not be 0). Pairs of one page with different n_valid
// share a tile: slots between theirs are multiplied by 0 for the shorter ones. Such a page is therefore planned twice, in
// tiles as any other and, behind all of these, with a tile for each of its pairs; the split looks over the rows of V that
// only some of its readers read, and the read takes the pairs one by one if a value there is not finite. Where all of 64
// pages of 512 slots differ in 4 (256) rows, 64 rows of top-4 routing take 108 (154) us in place of 81, 4096 rows 488 (495)
// in place of 481; with an infinity on each of them 214 (243) and 9500 (8400).
#pragma once

#include <math_constants.h>

#include "gemm_f16x3.cuh"
#include "prefill.cuh"

namespace xencb {

constexpr int RS_N = 64;          // N of both products: TERMS * MT
constexpr int RS_SEG = 512;       // slots of a unit
constexpr int RS_MAX_CS = 8;      // CTAs per cluster: 4, or 8
constexpr int RS_SLAB = 512;      // columns of d_s per CTA at most (4 x 64 TMEM columns)
constexpr int RS_VROWS = 48;      // slots per stage of the read
constexpr int RS_ACC = 4;         // score accumulators in TMEM
constexpr int RS_CHUNK = 2;       // TERMS = 2: k-blocks per accumulator (8 accumulation steps)
constexpr int RS_S_COL = 256;     // their first TMEM column (the read's sums lie below)
constexpr float RS_P_SCALE = 16384.f;     // P is scaled by 2^14
constexpr int RS_KTILE = 128 * 128;       // K tile of a stage: up to 128 slots x 64 columns; Q's 64 rows behind it
constexpr int RS_STAGE = RS_KTILE + RS_N * 128;  // scores; the read: 4 boxes of 48 slots x 64 columns
constexpr int RS_STAGES = 6;
constexpr int RS_PBLK = RS_N * 128;       // P of 64 slots: one 128-byte swizzle row per N row
constexpr int RS_STAT = 2 * 16 * RS_N;    // floats: [2][16 groups of 32 slots][MT]
constexpr int RS_SM_WARPS = 8;            // softmax: 4 TMEM lane quarters (32 slots each) x 2 halves of the pairs
constexpr int RS_FEW = 16;                // N rows of a unit whose read runs on the softmax warps
constexpr int RS_THREADS = 32 * 14;       // 0-7 softmax, 8-11 epilogue, 12 producer, 13 MMA
constexpr size_t RS_SMEM = 1024 + 8 * RS_PBLK + (size_t)RS_STAGES * RS_STAGE + 2 * RS_STAT * 4 +
                           (2 * RS_STAGES + 2 * RS_ACC + 9) * 8 + 16;
static_assert(RS_STAGES % 2 == 0, "a stage of V goes to the same four warps each time round the ring");
static_assert(4 * RS_VROWS * 128 <= RS_STAGE, "a stage of the read fits");

struct __align__(16) SharedTile {
  int page, start, count, nv;  // pairs [start, start + count) in grouped order; nv: their most valid slots
};
// flags beside `start` (there are fewer than 2^30 pairs) of a page whose readers disagree on n_valid: a tile of all of
// them, and one of a single pair
constexpr int RS_MIXED = 1 << 30, RS_SINGLE = -2147483647 - 1;

struct SharedArgs {
  // plan inputs
  const int32_t* page_of;   // [n_lib, C]
  const int32_t* n_valid;   // [n_lib, C]
  const int32_t* idx;       // [R, k]
  const float* wk;          // [R, k]
  int64_t n_rows, rows_per_lib, n_lib;
  int k, C, n_pages, page_rows, d_s;
  int n_pairs;
  // plan outputs (workspace)
  int* cnt;        // [n_pages]: pairs per page, then the page's first grouped position
  int* nvmax;      // [n_pages]
  int* page;       // [n_pairs]: page of a pair, -1: reads nothing
  int* rank;       // [n_pairs]: its place among the page's pairs; then its grouped position
  SharedTile* tiles;
  int* n_tiles;
  int* pnv;        // [n_pairs] by position: valid slots
  float* qinv;     // [n_pairs] by position: 1 / (the row's power-of-two scale)
  // read
  int segs, cs, ns, slab;  // segments of a page; CTAs per cluster, slots and columns of d_s per CTA
  int v3d;         // V's map is 3-D: [64 columns][slots][blocks of 64 columns] (d_s a multiple of 64)
  float qscale;    // read_temp * log2(e), or 1
  int softmax;
  float* part;     // [n_pairs][segs][d_s], normalised per segment
  float2* ml;      // [n_pairs][segs]: (max, sum)
  // pages whose readers disagree on n_valid ("mixed")
  int* nvgap;         // [n_pages]: page_rows less the page's fewest valid slots; after the split -1: not all finite
  int* n_mixed;       // their number; the number of their single tiles, which lie behind all others; 1: these are read
  int* mixed;         // [n_pages]: the mixed pages
  int* single;        // [n_pages]: the first of a mixed page's single tiles, -1: not mixed
  const uint16_t* v;  // the value pool's bits
  uint32_t v_exp;     // the exponent bits of its type
};

// ----------------------------------------------------------------------------------------------------- plan
__device__ __forceinline__ void rs_count(const SharedArgs& a, int64_t first, int64_t step) {
  for (int64_t i = first; i < a.n_pairs; i += step) {
    const int64_t row = i / a.k;
    const int64_t lib = row / a.rows_per_lib;
    const int c = a.idx[i];
    int page = -1;
    if (c >= 0 && a.wk[i] != 0.f) {
      if (c < a.C) page = a.page_of[lib * a.C + c];
      if (page < 0 || page >= a.n_pages) {
        flag_error(XENCB_DEV_BADPAGE);
        page = -1;
      }
    }
    if (page >= 0) {
      int nv = a.n_valid[lib * a.C + c];
      if (nv > a.page_rows) {
        nv = a.page_rows;
        flag_error(XENCB_DEV_CLAMPED);
      }
      if (nv <= 0) {
        page = -1;
      } else {
        a.rank[i] = atomicAdd(&a.cnt[page], 1);
        atomicMax(&a.nvmax[page], nv);
        if (nv < a.page_rows) atomicMax(&a.nvgap[page], a.page_rows - nv);
      }
    }
    a.page[i] = page;
  }
}

// One CTA of 1024 threads: positions of the pages' first pairs (into cnt) and the tiles of mt pairs.
__device__ __forceinline__ void rs_scan(const SharedArgs& a, int mt) {
  __shared__ int sh_pos[32], sh_tile[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int per = (a.n_pages + 1023) / 1024;
  const int p0 = min(a.n_pages, (int)threadIdx.x * per), p1 = min(a.n_pages, p0 + per);
  int pos = 0, tiles = 0;
  for (int p = p0; p < p1; ++p) {
    const int c = a.cnt[p];
    pos += c;
    tiles += (c + mt - 1) / mt;
  }
  int ip = pos, it = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int yp = __shfl_up_sync(0xffffffffu, ip, o), yt = __shfl_up_sync(0xffffffffu, it, o);
    if (lane >= o) { ip += yp; it += yt; }
  }
  if (lane == 31) { sh_pos[wid] = ip; sh_tile[wid] = it; }
  __syncthreads();
  int wp = sh_pos[lane], wt = sh_tile[lane];
  const int wp0 = wp, wt0 = wt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int yp = __shfl_up_sync(0xffffffffu, wp, o), yt = __shfl_up_sync(0xffffffffu, wt, o);
    if (lane >= o) { wp += yp; wt += yt; }
  }
  if (threadIdx.x == 1023) *a.n_tiles = wt;
  const int all = __shfl_sync(0xffffffffu, wt, 31);
  int at = ip - pos + __shfl_sync(0xffffffffu, wp - wp0, wid);
  int tile = it - tiles + __shfl_sync(0xffffffffu, wt - wt0, wid);
  for (int p = p0; p < p1; ++p) {
    const int c = a.cnt[p];
    a.cnt[p] = at;
    const int nv = a.nvmax[p];
    const bool mixed = nv > a.page_rows - a.nvgap[p];
    for (int s = 0; s < c; s += mt)
      a.tiles[tile++] = SharedTile{p, (at + s) | (mixed ? RS_MIXED : 0), min(mt, c - s), nv};
    if (mixed) a.mixed[atomicAdd(a.n_mixed, 1)] = p;
    a.single[p] = mixed ? all + atomicAdd(a.n_mixed + 1, c) : -1;  // (the split writes these tiles)
    at += c;
  }
}

__global__ void __launch_bounds__(256) shared_count_kernel(const SharedArgs a) {
  rs_count(a, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

__global__ void __launch_bounds__(1024) shared_scan_kernel(const SharedArgs a, int mt) {
  pdl_trigger();  // (the split reads q, which no kernel from here on writes, and waits before anything else)
  rs_scan(a, mt);
}

// Few pairs: the whole plan in one CTA.
__global__ void __launch_bounds__(1024) shared_plan_kernel(const SharedArgs a, int mt) {
  pdl_trigger();
  if (threadIdx.x < 3) a.n_mixed[threadIdx.x] = 0;
  for (int p = threadIdx.x; p < a.n_pages; p += 1024) {
    a.cnt[p] = 0;
    a.nvmax[p] = 0;
    a.nvgap[p] = 0;
  }
  __syncthreads();
  rs_count(a, threadIdx.x, 1024);
  __syncthreads();
  rs_scan(a, mt);
}

// Are the rows of V that only some readers of a mixed page read finite? The grid takes 16 rows at a time.
__device__ __forceinline__ void rs_check_mixed(const SharedArgs& a, int n, int threads) {
  const int per = (a.page_rows + 15) / 16;
  const int64_t step = (int64_t)gridDim.x * gridDim.y;
  for (int64_t w = (int64_t)blockIdx.y * gridDim.x + blockIdx.x; w < (int64_t)n * per; w += step) {
    const int page = a.mixed[w / per], gap = *reinterpret_cast<volatile int*>(&a.nvgap[page]);
    if (gap < 0) continue;  // (found already)
    const int lo = a.page_rows - gap + (int)(w % per) * 16, hi = min(lo + 16, a.nvmax[page]);
    const uint16_t* v = a.v + ((int64_t)page * a.page_rows + lo) * a.d_s;
    const uint32_t e0 = a.v_exp, e1 = a.v_exp << 16;
    bool bad = false;
#pragma unroll 4
    for (int i = (int)threadIdx.x * 8; i < (hi - lo) * a.d_s; i += threads * 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(v + i);
      const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= (x[e] & e0) == e0 || (x[e] & e1) == e1;
    }
    if (bad) {
      a.nvgap[page] = -1;
      a.n_mixed[2] = 1;
    }
  }
}

// Each pair's q row in 16 bits at the pair's grouped position: hi terms [n_pairs, d_s], then (TERMS = 2) lo terms. One
// CTA per row and up to 8 of its routed chunks; the row stays in registers (d_s <= 4096: two pieces of 8 a thread).
constexpr int RS_SPLIT_THREADS = 256;
template <typename TQ, typename T, int TERMS>
__global__ void __launch_bounds__(RS_SPLIT_THREADS, TERMS == 1 ? 8 : std::is_same<T, __half>::value ? 5 : 6)
    shared_split_kernel(const TQ* __restrict__ q, const SharedArgs a, T* __restrict__ out) {
  __shared__ float red[8];
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const TQ* src = q + row * a.d_s;
  float v[2][8];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int i = (p * RS_SPLIT_THREADS + threadIdx.x) * 8;
    if (i < a.d_s) load8_f32<TQ>(src + i, v[p]);
  }
  float s = 1.f;
  if (std::is_same<T, __half>::value) {  // f16's range: the row's largest value to [2^14, 2^15)
    float mx = 0.f;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      if ((p * RS_SPLIT_THREADS + threadIdx.x) * 8 < a.d_s)
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[p][e]));
    mx = warp_max(mx);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) mx = fmaxf(mx, red[w]);
    s = f16_range_scale(mx);
  }
  alignas(16) T hi[2][8], lo[2][8];
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[p][e] = from_f32<T>(v[p][e] * s);
      if (TERMS == 2) lo[p][e] = from_f32<T>(v[p][e] * s - to_f32(hi[p][e]));
    }
  pdl_wait();  // the plan
  const int n_mixed = *a.n_mixed;
  const int64_t lib = row / a.rows_per_lib;
  const int j1 = min(a.k, (int)(blockIdx.y + 1) * 8);
  for (int j = blockIdx.y * 8; j < j1; ++j) {
    const int64_t pair = row * a.k + j;
    const int page = a.page[pair];
    if (page < 0) continue;
    const int pos = a.cnt[page] + a.rank[pair];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int i = (p * RS_SPLIT_THREADS + threadIdx.x) * 8;
      if (i >= a.d_s) continue;
      *reinterpret_cast<uint4*>(out + (int64_t)pos * a.d_s + i) = *reinterpret_cast<const uint4*>(hi[p]);
      if (TERMS == 2)
        *reinterpret_cast<uint4*>(out + ((int64_t)a.n_pairs + pos) * a.d_s + i) =
            *reinterpret_cast<const uint4*>(lo[p]);
    }
    if (threadIdx.x == 0) {
      const int nv = min(a.n_valid[lib * a.C + a.idx[pair]], a.page_rows);
      a.pnv[pos] = nv;
      a.qinv[pos] = 1.f / s;
      const int single = n_mixed ? a.single[page] : -1;
      if (single >= 0) a.tiles[single + a.rank[pair]] = SharedTile{page, pos | RS_SINGLE, 1, nv};
    }
  }
  if (n_mixed) rs_check_mixed(a, n_mixed, RS_SPLIT_THREADS);
}

// ----------------------------------------------------------------------------------------------------- cluster PTX
// 3-D tiled TMA load (no multicast): the innermost coordinate must be 16-byte aligned.
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(smem_dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_3d_hint(void* smem_dst, const CUtensorMap* map, int x, int y, int z,
                                                 uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// True in one thread of a converged warp. The compiler issues TMA and MMA instructions of an elected thread from
// uniform registers; under `lane == 0` each cost about 150 cycles to issue, which bound the kernel (one stage of three
// copies 770 cycles, whatever its bytes).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "elect.sync _|P, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(p));
  return p != 0;
}
// A 4-byte store to a CTA of the cluster that counts its bytes on that CTA's barrier: the value and its arrival in one
// trip, where a store, a release and an arrival took 1 us more.
__device__ __forceinline__ void st_async_f32(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(addr),
               "r"(__float_as_uint(v)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait for a barrier that other CTAs of the cluster arrive on.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t it = 1;; ++it) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if ((it & 63u) == 0u && clock64() - t0 > XENCB_WAIT_CYCLES) {
      flag_error(XENCB_DEV_TIMEOUT);
      return false;
    }
  }
}
// Bulk copy from this CTA's shared memory to another CTA's, counted on that CTA's barrier. 16-byte units.
__device__ __forceinline__ void bulk_s2s(uint32_t dst_cluster, const void* src, uint32_t bytes, uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_cluster),
      "r"(smem_u32(src)), "r"(bytes), "r"(bar_cluster)
      : "memory");
}

// ----------------------------------------------------------------------------------------------------- read
struct RsSmem {
  unsigned char* p;       // [8 blocks of 64 slots][RS_PBLK]
  unsigned char* stages;  // the ring
  float* smax;            // [2][16][MT]: by the parity of the unit, per 32 slots
  float* ssum;            // [2][16][MT]
  // p_full and sums: [0] units whose read runs on the tensor core, [1] units of few pairs. Each has one set of waiters,
  // which sees every phase.
  uint64_t *full, *empty, *s_full, *s_empty, *p_full, *o_full, *o_empty, *stat, *sums, *seen, *v_done;
  uint32_t* tmem;
  volatile int* abort_flag;
};

// A place in the ring of stages: the stage and the parity of its next completion.
struct RsRing {
  uint32_t st, phase;
  __device__ __forceinline__ void next(uint32_t n) {
    if (++st == n) { st = 0; phase ^= 1; }
  }
  __device__ __forceinline__ void skip(uint32_t by, uint32_t n) {
    st += by;
    phase ^= (st / n) & 1;
    st %= n;
  }
  __device__ __forceinline__ void back(uint32_t n) {
    if (st == 0) { st = n; phase ^= 1; }
    --st;
  }
};

__device__ __forceinline__ RsSmem rs_smem(unsigned char* base) {
  RsSmem s;
  s.p = base;
  s.stages = base + 8 * RS_PBLK;
  s.smax = reinterpret_cast<float*>(s.stages + RS_STAGES * RS_STAGE);
  s.ssum = s.smax + RS_STAT;
  s.full = reinterpret_cast<uint64_t*>(s.ssum + RS_STAT);
  s.empty = s.full + RS_STAGES;
  s.s_full = s.empty + RS_STAGES;
  s.s_empty = s.s_full + RS_ACC;
  s.p_full = s.s_empty + RS_ACC;
  s.o_full = s.p_full + 2;
  s.o_empty = s.o_full + 1;
  s.stat = s.o_empty + 1;
  s.sums = s.stat + 1;
  s.seen = s.sums + 2;
  s.v_done = s.seen + 1;
  s.tmem = reinterpret_cast<uint32_t*>(s.v_done + 1);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem + 1);
  return s;
}

// A unit of this cluster: a tile and one segment of its page. Every warp walks the same list.
struct RsUnit {
  int u;  // >= n_units: none
  SharedTile t;
  int seg0, nv;  // first slot, valid slots (of the pair with most) in the segment
  __device__ __forceinline__ void find(const SharedArgs& a, int first, int n_units, int step) {
    for (u = first; u < n_units; u += step) {
      t = a.tiles[u / a.segs];
      if (t.start & (RS_MIXED | RS_SINGLE)) {  // one form or the other
        if ((a.nvgap[t.page] < 0) != ((t.start & RS_SINGLE) != 0)) continue;
        t.start &= ~(RS_MIXED | RS_SINGLE);
      }
      seg0 = (u % a.segs) * RS_SEG;
      nv = min(t.nv - seg0, RS_SEG);
      if (nv > 0) return;
    }
  }
};

// Reduction over a warp's 32 lanes of N values a lane (N = 16 or 32): lane l returns the reduced value l % N. Each
// step exchanges half of the values that are left: N - 1 shuffles (one more for N = 16) in place of 5 N.
template <int N, typename F>
__device__ __forceinline__ float rs_reduce(const float (&v)[N], int lane, F op) {
  float a[N];
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = v[i];
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? a[i] : a[i + o], keep = up ? a[i + o] : a[i];
      a[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  if (N == 16) a[0] = op(a[0], __shfl_xor_sync(0xffffffffu, a[0], 16));
  return a[0];
}

template <typename T, int TERMS>
__global__ void __launch_bounds__(RS_THREADS, 1)
    shared_read_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q8,
                       const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const SharedArgs a) {
  constexpr int MT = RS_N / TERMS;                    // pairs per tile
  constexpr int PP = MT / 2;                          // pairs of a softmax warp
  constexpr int FMT = std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16;
  extern __shared__ unsigned char rs_smem_raw[];
  const RsSmem s = rs_smem(reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(rs_smem_raw) + 1023) &
                                                            ~uintptr_t(1023)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = a.cs, ns = a.ns;
  const int rank = (int)cluster_rank();
  const int cluster = blockIdx.x / cs, n_clusters = gridDim.x / cs;
  const int nkb = (a.d_s + 63) / 64;
  const int kpc = TERMS == 2 ? RS_CHUNK : nkb;                     // k-blocks per score accumulator
  const int x0 = rank * a.slab;                                    // this CTA's columns of d_s
  const int my_boxes = max(0, min(a.slab, a.d_s - x0) + 63) / 64;  // in boxes of 64
  const int quarters = ns / 32;                                    // of the TMEM lanes hold slots
  const int sm_warps = 2 * quarters;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_q8);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    for (int i = 0; i < RS_STAGES; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < RS_ACC; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_empty[i], sm_warps);
    }
    mbar_init(&s.p_full[0], 1);
    mbar_init(&s.p_full[1], 1);
    mbar_init(s.o_full, 1);
    mbar_init(s.o_empty, 4);
    mbar_init(s.stat, 1);  // and the bytes of cs * sm_warps * PP values (sums too)
    mbar_init(&s.sums[0], 1);
    mbar_init(&s.sums[1], 1);
    mbar_init(s.seen, 4);
    mbar_init(s.v_done, RS_SM_WARPS + 1);  // and the MMA thread, so that it sees every phase
    *s.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 13) {
    tc_alloc(s.tmem, 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // every CTA's barriers exist before another CTA arrives on them
  tc_fence_after();
  const uint32_t taddr = *s.tmem;
  pdl_wait();
  const int n_units = (*a.n_tiles + (a.n_mixed[2] ? a.n_mixed[1] : 0)) * a.segs;
  RsUnit cur, nxt;
  cur.find(a, cluster, n_units, n_clusters);
  // few pairs: the read runs on the softmax warps (which are all there with 128 slots a CTA)
  auto is_few = [&](const RsUnit& w) { return w.t.count * TERMS <= RS_FEW && ns == 128; };
  auto s_stages = [&](const RsUnit& w) { return w.u < n_units && rank * ns < w.nv ? nkb : 0; };
  auto v_stages = [&](const RsUnit& w) { return (w.nv + RS_VROWS - 1) / RS_VROWS * ((my_boxes + 3) / 4); };
  // A wait that runs out sets the abort flag; from then on the softmax and epilogue warps wait for nothing and run
  // through their units on whatever is there, so that the named barrier stays matched.
  // The lanes of a warp may leave a wait one after the other: they meet again here, as the tensor-memory loads, mma.sync,
  // ldmatrix and barriers that follow need a converged warp.
  auto done = [&](bool arrived) {
    if (!arrived) *s.abort_flag = 1;
    __syncwarp();
  };

  if (warp == 12) {
    // --------------------------------------------------------------------------------------------- producer
    if (elect_one()) {
      // The clusters hold a page each that is to be read again and one that is arriving, about the size of L2: K's
      // lines are kept, V's pass (the second of a tied page) lets them go.
      const uint64_t keep = policy_evict_last(), let_go = policy_evict_first();
      RsRing ring{0, 0};
      uint32_t used = 0;
      bool ok = true;
      auto scores = [&](const RsUnit& w) {
        if (w.u >= n_units || rank * ns >= w.nv) return;
        const int y = w.t.page * a.page_rows + w.seg0 + rank * ns;
        const bool few = w.t.count <= 8;  // eight rows of Q a term; what lies in the others is not looked at
        const uint32_t tx = (uint32_t)((few ? 8 : MT) * TERMS + ns) * 128;
        for (int kb = 0; kb < nkb && ok; ++kb) {
          if (used >= RS_STAGES) ok = mbar_wait_spin(&s.empty[ring.st], ring.phase ^ 1);
          if (!ok) break;
          uint64_t* bar = &s.full[ring.st];
          unsigned char* st = s.stages + ring.st * RS_STAGE;
          mbar_arrive_expect_tx(bar, tx);
          tma_load_2d_hint(st, &map_k, kb * 64, y, bar, keep);
          if (few) {
#pragma unroll
            for (int x = 0; x < TERMS; ++x)
              tma_load_2d(st + RS_KTILE + x * MT * 128, &map_q8, kb * 64, x * a.n_pairs + w.t.start, bar);
          } else {
            tma_load_3d(st + RS_KTILE, &map_q, kb * 64, w.t.start, 0, bar);
          }
          ring.next(RS_STAGES);
          ++used;
        }
      };
      auto values = [&](const RsUnit& w) {
        const int y = w.t.page * a.page_rows + w.seg0;
        for (int b = 0; b < (w.nv + RS_VROWS - 1) / RS_VROWS && ok; ++b)
          for (int h = 0; h < my_boxes; h += 4) {
            const int n = min(4, my_boxes - h);
            if (used >= RS_STAGES) ok = mbar_wait_spin(&s.empty[ring.st], ring.phase ^ 1);
            if (!ok) break;
            uint64_t* bar = &s.full[ring.st];
            unsigned char* st = s.stages + ring.st * RS_STAGE;
            mbar_arrive_expect_tx(bar, (uint32_t)(a.v3d ? 4 : n) * RS_VROWS * 128);
            if (a.v3d)  // four boxes of 64 columns in one copy (those past d_s arrive as zeros)
              tma_load_3d_hint(st, &map_v, 0, y + b * RS_VROWS, (x0 >> 6) + h, bar, let_go);
            else
              for (int i = 0; i < n; ++i)
                tma_load_2d_hint(st + i * RS_VROWS * 128, &map_v, x0 + (h + i) * 64, y + b * RS_VROWS, bar, let_go);
            ring.next(RS_STAGES);
            ++used;
          }
      };
      scores(cur);
      while (cur.u < n_units && ok) {
        nxt.find(a, cur.u + n_clusters, n_units, n_clusters);
        scores(nxt);
        values(cur);
        cur = nxt;
      }
      if (!ok) *s.abort_flag = 1;
      // the copies in flight end before the CTA's shared memory goes away
      for (uint32_t i = min(used, (uint32_t)RS_STAGES); i > 0; --i) {
        ring.back(RS_STAGES);
        mbar_wait_bounded(&s.full[ring.st], ring.phase);
      }
    }
    __syncwarp();
  } else if (warp == 13) {
    // --------------------------------------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      RsRing ring{0, 0};
      uint32_t big = 0, few = 0, acc = 0;  // units whose read runs here, and on the softmax warps
      bool ok = true;
      const uint32_t id_s = umma_idesc(FMT, FMT, 128, RS_N);
      const uint32_t id_o = umma_idesc(FMT, FMT, 128, RS_N) | (1u << 15);  // A (V) is MN-major
      // operand descriptors: the constant part, and addresses in 16-byte units (14 bits: the address of a CTA's shared
      // memory carries its cluster rank above them)
      const uint64_t dk = umma_desc_k_sw128(0), dv = umma_desc_mn_sw128(0, RS_VROWS * 128);
      const uint32_t st0 = (smem_u32(s.stages) >> 4) & 0x3FFFu, p0 = (smem_u32(s.p) >> 4) & 0x3FFFu;
      auto scores = [&](const RsUnit& w) {
        if (w.u >= n_units || rank * ns >= w.nv) return;
        for (int k0 = 0; k0 < nkb && ok; k0 += kpc, ++acc) {
          const uint32_t buf = acc % RS_ACC, use = acc / RS_ACC;
          if (use > 0 && !(ok = mbar_wait_spin(&s.s_empty[buf], (use - 1) & 1))) break;
          tc_fence_after();
          const int k1 = min(nkb, k0 + kpc);
          for (int kb = k0; kb < k1; ++kb) {
            if (!(ok = mbar_wait_spin(&s.full[ring.st], ring.phase))) break;
            tc_fence_after();
            const uint64_t da = dk + (st0 + ring.st * (RS_STAGE / 16)), db = da + RS_KTILE / 16;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc_mma<0>(taddr + RS_S_COL + buf * RS_N, da + ks * 2, db + ks * 2, id_s, kb > k0 || ks > 0);
            tc_commit(&s.empty[ring.st]);
            ring.next(RS_STAGES);
          }
          if (!ok) break;
          tc_commit(&s.s_full[buf]);
        }
      };
      auto values = [&](const RsUnit& w) {
        for (int b = 0; b < (w.nv + RS_VROWS - 1) / RS_VROWS && ok; ++b) {
          const int left = w.nv - b * RS_VROWS, steps = min(RS_VROWS / 16, (left + 15) / 16);
          for (int h = 0; h < my_boxes; h += 4) {
            const int n = min(4, my_boxes - h);
            if (!(ok = mbar_wait_spin(&s.full[ring.st], ring.phase))) break;
            tc_fence_after();
            if (left < steps * 16) {  // rows of V behind the last valid slot: zeros (0 * NaN would not be 0)
              unsigned char* base = s.stages + ring.st * RS_STAGE;
              for (int i = 0; i < n; ++i)
                for (int c = left * 8; c < steps * 16 * 8; ++c)
                  *reinterpret_cast<uint4*>(base + i * RS_VROWS * 128 + c * 16) = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
            }
            const uint64_t dx = dv + (st0 + ring.st * (RS_STAGE / 16));
            for (int ks = 0; ks < steps; ++ks) {
              const int slot = b * RS_VROWS + ks * 16;  // its 16 slots of P lie in one block of 64
              const uint64_t dp = dk + (p0 + (slot >> 6) * (RS_PBLK / 16) + ((slot & 63) >> 3));
              // columns [128 t, 128 t + 128) of the slab: two boxes (the second may be stale: lanes nobody reads)
              for (int t = 0; t < (n + 1) / 2; ++t)
                tc_mma<0>(taddr + (uint32_t)(h / 2 + t) * RS_N, dx + t * (2 * RS_VROWS * 128 / 16) + ks * 128, dp, id_o,
                          b > 0 || ks > 0);
            }
            tc_commit(&s.empty[ring.st]);
            ring.next(RS_STAGES);
          }
        }
        if (ok) tc_commit(s.o_full);
      };
      scores(cur);
      while (cur.u < n_units && ok) {
        nxt.find(a, cur.u + n_clusters, n_units, n_clusters);
        scores(nxt);
        if (is_few(cur)) {
          // the softmax warps take these stages: a wait for a later use of a stage is one for a parity, so it may only
          // begin when every use before it is complete
          mbar_arrive(s.v_done);
          if (ok) ok = mbar_wait_spin(s.v_done, few & 1);
          ++few;
          ring.skip(v_stages(cur), RS_STAGES);
        } else {
          // the epilogue of the last such unit has read its sums, and every CTA's block of P is here
          if (ok && big > 0) ok = mbar_wait_spin(s.o_empty, (big - 1) & 1);
          if (ok) ok = mbar_wait_cluster(&s.p_full[0], big & 1);
          tc_fence_after();
          if (ok) values(cur);
          ++big;
        }
        cur = nxt;
      }
      if (!ok) *s.abort_flag = 1;
    }
    __syncwarp();
  } else if (warp < RS_SM_WARPS) {
    // --------------------------------------------------------------------------------------------- softmax
    // Lane = slot, registers = this warp's pairs.
    const int quarter = warp & 3, half = warp >> 2;
    if (quarter < quarters) {
      const uint32_t tl = taddr + ((uint32_t)(quarter * 32) << 16) + RS_S_COL + (uint32_t)(half * PP);
      const int slot0 = rank * ns + quarter * 32;              // lane 0's slot of the segment
      const int nth_warp = half * quarters + quarter;          // of the sm_warps
      const int group = slot0 >> 5;                            // 32 slots: their entry of smax and ssum
      // P: this CTA's block of the slot; 16-byte chunk j of row r at chunk j ^ (r % 8)
      const int in_blk = (quarter * 32 + lane) & 63;
      unsigned char* const pcol = s.p + (size_t)(rank * (ns / 64) + (quarter >> 1)) * RS_PBLK + (in_blk & 7) * 2;
      uint32_t unit = 0, big = 0, acc = 0;
      bool was_big = false;
      RsRing ring{0, 0};
      float v[PP];
      auto scores = [&](const RsUnit& w) {
        if (w.u >= n_units || rank * ns >= w.nv) return;
        for (int k0 = 0; k0 < nkb; k0 += kpc, ++acc) {
          const uint32_t buf = acc % RS_ACC;
          done(*s.abort_flag || mbar_wait_spin(&s.s_full[buf], (acc / RS_ACC) & 1));
          tc_fence_after();
          float x[PP];
          if constexpr (TERMS == 2) {
            float y[PP];
            tc_ld16(tl + buf * RS_N, x);
            tc_ld16(tl + buf * RS_N + MT, y);
#pragma unroll
            for (int i = 0; i < PP; ++i) x[i] += y[i];
          } else {
            tc_ld32(tl + buf * RS_N, x);
          }
#pragma unroll
          for (int i = 0; i < PP; ++i) v[i] = k0 == 0 ? x[i] : v[i] + x[i];
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.s_empty[buf]);
          __syncwarp();
        }
      };
      // The read of a unit of few pairs: O^T[64 columns, N] of this warp = V^T . P^T with N = 8 or 16: four pairs' hi rows
      // and their lo rows (TERMS = 2) or 8 pairs to a tile of 8. Warp w takes the w-th 64 columns of the slab; the four
      // warps of a stage hand it back together. mma.sync bounds it (a tile of 16 x 8 x 16 takes 32 cycles of a
      // scheduler; 18k cycles a unit of 512 slots): the columns as its 16 rows need half the products that the pairs as its
      // rows did.
      auto read_few = [&](const RsUnit& w, uint32_t un, uint32_t nth, RsRing rg) {
        done(*s.abort_flag || mbar_wait_cluster(&s.p_full[1], nth & 1));
        const int hgroups = (my_boxes + 3) / 4, hg = warp >> 2;
        if (hg >= hgroups) {  // no columns: but every phase of the barriers is waited for
          done(*s.abort_flag || mbar_wait_cluster(&s.sums[1], nth & 1));
          if (lane == 0) mbar_arrive(s.v_done);
          return;
        }
        const bool two = w.t.count * TERMS > 8;
        const int mtx = lane >> 3, r8 = lane & 7;
        // P: matrices (tile 0, slots 0-7), (tile 0, 8-15), (tile 1, 0-7), (tile 1, 8-15); row r8 of a tile
        const int pair_of = TERMS == 2 ? (mtx >> 1) * 4 + (r8 & 3) : (mtx >> 1) * 8 + r8;
        const int prow = TERMS == 2 ? (r8 >> 2) * MT + pair_of : pair_of;
        const uint32_t pa = smem_u32(s.p) + prow * 128;
        // V: matrices (slots 0-7, columns 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15), transposed
        const uint32_t vrow = (uint32_t)(warp & 3) * (RS_VROWS * 128) + (r8 + (mtx >> 1) * 8) * 128;
        float acc_o[4][2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) acc_o[i][x][0] = acc_o[i][x][1] = acc_o[i][x][2] = acc_o[i][x][3] = 0.f;
        rg.skip(hg, RS_STAGES);
        for (int b = 0; b < (w.nv + RS_VROWS - 1) / RS_VROWS; ++b) {
          done(*s.abort_flag || mbar_wait_spin(&s.full[rg.st], rg.phase));
          const uint32_t va = smem_u32(s.stages) + rg.st * RS_STAGE + vrow;
          const int left = w.nv - b * RS_VROWS;
#pragma unroll
          for (int ks = 0; ks < RS_VROWS / 16; ++ks) {
            if (ks * 16 >= left) break;
            const int slot = b * RS_VROWS + ks * 16;
            uint32_t p[4];
            ldsm_x4(pa + (slot >> 6) * RS_PBLK + (((((slot & 63) >> 3) + (mtx & 1)) ^ (prow & 7)) << 4), p[0], p[1],
                    p[2], p[3]);
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;  // rows of V behind the last valid slot: zeros
            const int over = left - ks * 16;
            if (over < 16) {
              const int k = (lane & 3) * 2;
              keep0 = (k < over ? 0xffffu : 0u) | (k + 1 < over ? 0xffff0000u : 0u);
              keep1 = (k + 8 < over ? 0xffffu : 0u) | (k + 9 < over ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              uint32_t a0, a1, a2, a3;
              ldsm_x4_t(va + ks * 2048 + (((m * 2 + (mtx & 1)) ^ r8) << 4), a0, a1, a2, a3);
              a0 &= keep0; a1 &= keep0; a2 &= keep1; a3 &= keep1;
              mma16816<T>(acc_o[m][0], a0, a1, a2, a3, p[0], p[1]);
              if (two) mma16816<T>(acc_o[m][1], a0, a1, a2, a3, p[2], p[3]);
            }
          }
          __syncwarp();
          named_bar_sync(2 + hg, 128);
          if ((warp & 3) == 0 && lane == 0 && !*s.abort_flag) mbar_arrive(&s.empty[rg.st]);
          __syncwarp();
          rg.skip(hgroups, RS_STAGES);
        }
        if (lane == 0) mbar_arrive(s.v_done);
        done(*s.abort_flag || mbar_wait_cluster(&s.sums[1], nth & 1));
        const int seg = w.u % a.segs;
        const float* smax = s.smax + (un & 1) * 16 * MT;
        const float* ssum = s.ssum + (un & 1) * 16 * MT;
        // lane i: pair i's coefficient
        float coef = 0.f;
        if (lane < w.t.count) {
          float m = a.softmax ? -CUDART_INF_F : 0.f, l = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            m = fmaxf(m, smax[e * MT + lane]);
            l += ssum[e * MT + lane];
          }
          const int64_t pos = w.t.start + lane;
          if (a.softmax) coef = l != 0.f ? 1.f / l : 0.f;
          else coef = rsqrtf((float)a.pnv[pos]) / f16_range_scale(m);
          if (rank == 0 && warp == 0) a.ml[pos * a.segs + seg] = make_float2(m, l);
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (x == 1 && !two) break;
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // this lane's N = 2 (lane % 4) + e
            const int n = (lane & 3) * 2 + e;
            const int pr = TERMS == 2 ? x * 4 + (n & 3) : x * 8 + n;
            const float ci = __shfl_sync(0xffffffffu, coef, pr);
            float* dst = a.part + ((int64_t)(w.t.start + pr) * a.segs + seg) * a.d_s + x0;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              float lo = acc_o[m][x][e], hi = acc_o[m][x][2 + e];  // columns (lane / 4) and 8 further
              if (TERMS == 2) {  // the lo rows' parts lie two lanes further
                lo += __shfl_xor_sync(0xffffffffu, lo, 2);
                hi += __shfl_xor_sync(0xffffffffu, hi, 2);
              }
              const int c = warp * 64 + m * 16 + (lane >> 2);
              if (pr < w.t.count && (TERMS == 1 || (lane & 2) == 0)) {
                if (c < a.slab && x0 + c < a.d_s) dst[c] = lo * ci;
                if (c + 8 < a.slab && x0 + c + 8 < a.d_s) dst[c + 8] = hi * ci;
              }
            }
          }
        }
      };
      scores(cur);
      ring.skip(s_stages(cur), RS_STAGES);
      while (cur.u < n_units) {
        nxt.find(a, cur.u + n_clusters, n_units, n_clusters);
        const SharedTile t = cur.t;
        const bool mine = rank * ns < cur.nv;
        const bool few = is_few(cur);
        const int count = t.count - half * PP;                 // this warp's pairs of the tile (may be <= 0)
        float* smax = s.smax + (unit & 1) * 16 * MT + half * PP;
        float* ssum = s.ssum + (unit & 1) * 16 * MT + half * PP;
        // lane i holds pair i's valid slots (from this warp's first) and scale
        const int me = lane & (PP - 1);
        const int pos = t.start + half * PP + me;
        const int lim = me < count ? a.pnv[pos] - cur.seg0 - slot0 : 0;
        const float c = me < count ? a.qinv[pos] * a.qscale : 0.f;
        // t = scores * scale; masked slots -inf (softmax) or 0 (linear read). A pair whose every score is masked gets max
        // -inf and then NaN weights: it has no slot in this segment, so nothing reads them.
        const float none = a.softmax ? -CUDART_INF_F : 0.f;
        float mx = none;
        if (mine) {
          float w[PP];
#pragma unroll
          for (int i = 0; i < PP; ++i) {
            const float ci = __shfl_sync(0xffffffffu, c, i);
            const int li = __shfl_sync(0xffffffffu, lim, i);
            v[i] = lane < li ? v[i] * ci : none;
            w[i] = a.softmax ? v[i] : fabsf(v[i]);
          }
          mx = rs_reduce<PP>(w, lane, [](float p, float q) { return fmaxf(p, q); });
        }
        // the read of the unit before is done with P, and its epilogue with the maxima and sums two units back
        if (was_big) {
          done(*s.abort_flag || mbar_wait_spin(s.o_full, (big - 1) & 1));
          done(*s.abort_flag || mbar_wait_spin(s.seen, (big - 1) & 1));
        }
        // the pairs' maxima over these 32 slots to every CTA of the cluster
        const uint32_t stat_bytes = (uint32_t)(cs * sm_warps * PP * 4);
        if (nth_warp == 0 && lane == 0) mbar_arrive_expect_tx(s.stat, stat_bytes);
        if (lane < PP)
          for (int r = 0; r < cs; ++r)
            st_async_f32(cluster_map(&smax[group * MT + lane], r), mx, cluster_map(s.stat, r));
        done(*s.abort_flag || mbar_wait_cluster(s.stat, unit & 1));
        float l = 0.f;
        if (mine) {
          float m = none;
#pragma unroll
          for (int g = 0; g < 16; ++g) m = fmaxf(m, smax[g * MT + me]);
          const float ml = a.softmax ? m : f16_range_scale(m);
#pragma unroll
          for (int g = 0; g < PP; g += 8) {
            if (g >= count) break;
#pragma unroll
            for (int i = g; i < g + 8; ++i) {  // (rows behind the last pair are written and not looked at)
              const float mi = __shfl_sync(0xffffffffu, ml, i);
              v[i] = a.softmax ? RS_P_SCALE * pf_exp2(v[i] - mi) : v[i] * mi;
              const int r = half * PP + i;
              unsigned char* at = pcol + r * 128 + (((in_blk >> 3) ^ (r & 7)) << 4);
              const T hi = from_f32<T>(v[i]);
              *reinterpret_cast<T*>(at) = hi;
              if (TERMS == 2) *reinterpret_cast<T*>(at + MT * 128) = from_f32<T>(v[i] - to_f32(hi));
            }
          }
          fence_proxy_async_smem();
          if (a.softmax) l = rs_reduce<PP>(v, lane, [](float p, float q) { return p + q; });
        }
        __syncwarp();
        named_bar_sync(1, 32 * sm_warps);
        if (elect_one()) {
          const uint32_t bytes = (uint32_t)(ns / 64) * RS_PBLK;
          if (nth_warp == 0) {
            // the other CTAs' blocks and sums are still to come
            const int n_work = min(cs, (cur.nv + ns - 1) / ns);
            mbar_arrive_expect_tx(&s.p_full[few], (uint32_t)(n_work - (mine ? 1 : 0)) * bytes);
            mbar_arrive_expect_tx(&s.sums[few], stat_bytes);
          }
          // this CTA's block to the others: each warp takes every sm_warps-th of them
          unsigned char* src = s.p + (size_t)rank * bytes;
          if (mine && !*s.abort_flag)
            for (int r = nth_warp; r < cs; r += sm_warps)
              if (r > 0) {
                const uint32_t to = (uint32_t)((rank + r) % cs);
                bulk_s2s(cluster_map(src, to), src, bytes, cluster_map(&s.p_full[few], to));
              }
        }
        __syncwarp();
        if (lane < PP)
          for (int r = 0; r < cs; ++r)
            st_async_f32(cluster_map(&ssum[group * MT + lane], r), l, cluster_map(&s.sums[few], r));
        __syncwarp();
        ring.skip(s_stages(nxt), RS_STAGES);
        scores(nxt);  // (and with them every stage before this unit's V has been used: see v_done)
        if (few) read_few(cur, unit, unit - big, ring);
        else ++big;
        ring.skip(v_stages(cur), RS_STAGES);
        was_big = !few;
        ++unit;
        cur = nxt;
      }
    }
  } else {
    // --------------------------------------------------------------------------------------------- epilogue
    // Lane = column of d_s, registers = pairs.
    const int quarter = warp & 3;
    uint32_t unit = 0, big = 0;
    while (cur.u < n_units) {
      nxt.find(a, cur.u + n_clusters, n_units, n_clusters);
      const SharedTile t = cur.t;
      const int seg = cur.u % a.segs;
      if (is_few(cur)) {
        ++unit;
        cur = nxt;
        continue;
      }
      const float* smax = s.smax + (unit & 1) * 16 * MT;
      const float* ssum = s.ssum + (unit & 1) * 16 * MT;
      done(*s.abort_flag || mbar_wait_cluster(&s.sums[0], big & 1));
      float coef[MT / 32];  // lane i: pairs i and (TERMS = 1) 32 + i
#pragma unroll
      for (int g = 0; g < MT / 32; ++g) {
        const int i = g * 32 + lane;
        float m = a.softmax ? -CUDART_INF_F : 0.f, l = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          m = fmaxf(m, smax[e * MT + i]);
          l += ssum[e * MT + i];
        }
        coef[g] = 0.f;
        if (i < t.count) {
          const int64_t pos = t.start + i;
          if (a.softmax) coef[g] = l != 0.f ? 1.f / l : 0.f;
          else coef[g] = rsqrtf((float)a.pnv[pos]) / f16_range_scale(m);
          if (rank == 0 && warp == 8) a.ml[pos * a.segs + seg] = make_float2(m, l);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(s.seen);
      __syncwarp();
      done(*s.abort_flag || mbar_wait_spin(s.o_full, big & 1));
      tc_fence_after();
      for (int b = 0; b < (my_boxes + 1) / 2; ++b) {
        const int x = b * 128 + quarter * 32 + lane;  // column of the slab
        const bool in = x < a.slab && x0 + x < a.d_s;
        const int64_t pair_stride = (int64_t)a.segs * a.d_s;
        float* dst = a.part + ((int64_t)t.start * a.segs + seg) * a.d_s + x0 + x;
        const uint32_t at = taddr + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * RS_N);
#pragma unroll
        for (int g = 0; g < MT / 32; ++g) {
          if (g * 32 >= t.count) break;
          float o[32];
          tc_ld32(at + g * 32, o);
          if constexpr (TERMS == 2) {
            float y[32];
            tc_ld32(at + 32, y);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] += y[i];
          }
          float* d = dst + (int64_t)(g * 32) * pair_stride;
#pragma unroll
          for (int i8 = 0; i8 < 32; i8 += 8) {
            if (g * 32 + i8 >= t.count) break;
#pragma unroll
            for (int i = i8; i < i8 + 8; ++i, d += pair_stride) {
              const float x = o[i] * __shfl_sync(0xffffffffu, coef[g], i);
              if (in && g * 32 + i < t.count) *d = x;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s.o_empty);
      ++big;
      ++unit;
      cur = nxt;
    }
  }
  __syncwarp();
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while another may still write to its shared memory
  tc_fence_after();
  if (warp == 13) tc_dealloc(taddr, 512);
}

// ----------------------------------------------------------------------------------------------------- combine
// r[row] = sum_j wk[row, j] * (the pair's segments, merged by their maxima and sums). G groups of threads take the
// routed chunks j = group, group + G, ..., and their sums are added in the order of the groups, so the result depends
// on nothing but the row. G = 1 for up to 8 routed chunks (256 threads, 1024 columns), else 8 (128 columns).
template <typename TO, int G>
__global__ void __launch_bounds__(256) shared_combine_kernel(const SharedArgs a, TO* __restrict__ r) {
  constexpr int W = 256 / G;
  __shared__ float4 sum[G > 1 ? G : 1][G > 1 ? W : 1];
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int64_t lib = row / a.rows_per_lib;
  const int lane = threadIdx.x % W, grp = threadIdx.x / W;
  const int x = (blockIdx.y * W + lane) * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int j = grp; j < a.k; j += G) {
    const int64_t pair = row * a.k + j;
    const int page = a.page[pair];
    if (page < 0) continue;
    const int64_t pos = a.cnt[page] + a.rank[pair];
    const float w = a.wk[pair];
    const float* p = a.part + pos * a.segs * a.d_s + x;
    int segs = 1;
    float m = -CUDART_INF_F, z = 0.f;
    if (a.segs > 1) {
      const int nv = min(a.n_valid[lib * a.C + a.idx[pair]], a.page_rows);
      segs = (nv + RS_SEG - 1) / RS_SEG;
      if (a.softmax) {
        for (int g = 0; g < segs; ++g) m = fmaxf(m, a.ml[pos * a.segs + g].x);
        for (int g = 0; g < segs; ++g) {
          const float2 ml = a.ml[pos * a.segs + g];
          z += exp2f(ml.x - m) * ml.y;
        }
      }
    }
    for (int g = 0; g < segs; ++g) {
      float f = w;
      if (a.softmax && a.segs > 1) {
        const float2 ml = a.ml[pos * a.segs + g];
        f *= exp2f(ml.x - m) * ml.y / z;
      }
      if (x < a.d_s) {
        const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)g * a.d_s);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
    }
  }
  if (G > 1) {
    sum[grp][lane] = acc;
    __syncthreads();
    if (grp != 0) return;
#pragma unroll
    for (int g = 1; g < G; ++g) {
      const float4 v = sum[g][lane];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
  }
  if (x >= a.d_s) return;
  alignas(16) TO o[4] = {from_f32<TO>(acc.x), from_f32<TO>(acc.y), from_f32<TO>(acc.z), from_f32<TO>(acc.w)};
  if (sizeof(TO) == 4) *reinterpret_cast<uint4*>(r + row * a.d_s + x) = *reinterpret_cast<const uint4*>(o);
  else *reinterpret_cast<uint2*>(r + row * a.d_s + x) = *reinterpret_cast<const uint2*>(o);
}

}  // namespace xencb
