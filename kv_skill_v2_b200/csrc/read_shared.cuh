// Shared read: the routed two-level read (xenc/injector.py:239-265) with every page fetched once for ALL query rows
// that read it, whichever Libraries they belong to: forked Libraries whose tables name the same pages, many requests
// on one document, prompts with top-k routing.
//
//   r[t] = sum_j wk[t, j] * softmax_n(read_temp * q_t . K_p[n]) @ V_p,   p = page_of[lib(t), idx[t, j]], n < n_valid
//
// The (row, routed chunk) pairs are grouped by page (count, scan, scatter); a tile is one page with up to MT of its
// pairs, a unit one tile with up to 128 * cs of the page's slots. A cluster of cs CTAs computes a unit on the 5th
// generation tensor cores:
//   scores  CTA j: S[pairs, its slots] = Q . K^T over all of d_s (TMA tiles, f32 in TMEM);
//   softmax rows' maxima exchanged through distributed shared memory, P = 2^(t - max) in 16 bits, CTA j's block of P
//           sent to every CTA of the cluster (bulk copies between their shared memories, counted on an mbarrier);
//   read    CTA j: O[pairs, its columns of d_s] = P . V (V as an MN-major operand), scaled by 1 / sum, stored per pair.
// The scores and the read walk the page differently (all columns of some slots, all slots of some columns), so the page
// passes through shared memory twice, but its second pass comes from L2: a cluster holds one page at a time.
// shared_combine adds a row's pairs in the order of its routing: results do not depend on how pairs were grouped.
//
// Precision. The operands are 16-bit. TERMS = 2 (float32 outputs): q and P enter as hi + lo pairs stacked in the rows
// of one MMA (hi above lo: the same instructions cover both), which keeps 22 bits with f16 slots and 16 with bf16;
// the rows' halves are added in float32. TERMS = 1 (16-bit outputs): one rounding of q and of P, as the other
// tensor-core reads do. q is scaled by a power of two per row and P by 2^14, so f16's range is no limit.
//
// The tensor core's accumulator drops bits below its running value at every 16-term step, always towards zero; over
// d_s = 2048 that is 128 steps, 1.2e-5 of a score near 1, which read_temp multiplies. With TERMS = 2 the scores are
// therefore accumulated 128 columns of d_s at a time into a ring of TMEM buffers and added up in float32 registers.
//
// Slots at or past n_valid never reach a result: their scores are masked, P is 0 there, and the rows of V behind the
// tile's last valid slot are zeroed in shared memory (0 * NaN would not be 0).
#pragma once

#include <math_constants.h>

#include "gemm_f16x3.cuh"
#include "prefill.cuh"

namespace xencb {

constexpr int RS_AROWS = 64;      // rows of the A operands that carry data (TERMS * MT); the MMA's M is 128
constexpr int RS_MAX_CS = 8;      // CTAs per cluster: 4 (d_s <= 2048) or 8
constexpr int RS_SLAB = 512;      // columns of d_s per CTA at most (TMEM)
constexpr int RS_STAGES = 4;
constexpr int RS_STAGE = 32768;   // scores: A 8 KB + B 16 KB; read: 4 boxes of 64 slots x 64 columns
constexpr int RS_PBLK = RS_AROWS * 128;       // P of 64 slots: one 128-byte swizzle row per pair
constexpr int RS_THREADS = 32 * 10;           // producer, MMA, 8 softmax / epilogue warps
constexpr int RS_ACC = 4;         // score accumulators in TMEM (ns columns each)
constexpr int RS_CHUNK = 2;       // TERMS = 2: k-blocks per accumulator (8 accumulation steps)
constexpr float RS_P_SCALE = 16384.f;         // P is scaled by 2^14

struct __align__(16) SharedTile {
  int page, start, count, nv;  // pairs [start, start + count) in grouped order; nv: the page's most valid slots
};

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
  int segs, seg_rows, cs, ns, slab;
  float qscale;    // read_temp * log2(e), or 1
  int softmax;
  float* part;     // [n_pairs][segs][d_s], normalised per segment
  float2* ml;      // [n_pairs][segs]: (max, sum)
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
  int at = ip - pos + __shfl_sync(0xffffffffu, wp - wp0, wid);
  int tile = it - tiles + __shfl_sync(0xffffffffu, wt - wt0, wid);
  for (int p = p0; p < p1; ++p) {
    const int c = a.cnt[p];
    a.cnt[p] = at;
    for (int s = 0; s < c; s += mt) a.tiles[tile++] = SharedTile{p, at + s, min(mt, c - s), a.nvmax[p]};
    at += c;
  }
}

__global__ void __launch_bounds__(256) shared_count_kernel(const SharedArgs a) {
  rs_count(a, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

__global__ void __launch_bounds__(1024) shared_scan_kernel(const SharedArgs a, int mt) { rs_scan(a, mt); }

// Few pairs: the whole plan in one CTA.
__global__ void __launch_bounds__(1024) shared_plan_kernel(const SharedArgs a, int mt) {
  for (int p = threadIdx.x; p < a.n_pages; p += 1024) {
    a.cnt[p] = 0;
    a.nvmax[p] = 0;
  }
  __syncthreads();
  rs_count(a, threadIdx.x, 1024);
  __syncthreads();
  rs_scan(a, mt);
}

// Each pair's q row in 16 bits at the pair's grouped position: hi terms [n_pairs, d_s], then (TERMS = 2) lo terms.
template <typename TQ, typename T, int TERMS>
__global__ void __launch_bounds__(256) shared_split_kernel(const TQ* __restrict__ q, const SharedArgs a,
                                                           T* __restrict__ out) {
  __shared__ float red[8];
  const int64_t pair = blockIdx.x;
  const int page = a.page[pair];
  if (page < 0) return;
  const int64_t row = pair / a.k;
  const int pos = a.cnt[page] + a.rank[pair];
  const TQ* src = q + row * a.d_s;
  float s = 1.f;
  if (sizeof(T) == 2 && std::is_same<T, __half>::value) {  // f16's range: the row's largest value to [2^14, 2^15)
    float mx = 0.f;
    for (int i = threadIdx.x * 8; i < a.d_s; i += 256 * 8) {
      float v[8];
      load8_f32<TQ>(src + i, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e]));
    }
    mx = warp_max(mx);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) mx = fmaxf(mx, red[w]);
    s = f16_range_scale(mx);
  }
  for (int i = threadIdx.x * 8; i < a.d_s; i += 256 * 8) {
    float v[8];
    load8_f32<TQ>(src + i, v);
    alignas(16) T hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = from_f32<T>(v[e] * s);
      lo[e] = from_f32<T>(v[e] * s - to_f32(hi[e]));
    }
    *reinterpret_cast<uint4*>(out + (int64_t)pos * a.d_s + i) = *reinterpret_cast<const uint4*>(hi);
    if (TERMS == 2)
      *reinterpret_cast<uint4*>(out + ((int64_t)a.n_pairs + pos) * a.d_s + i) = *reinterpret_cast<const uint4*>(lo);
  }
  if (threadIdx.x == 0) {
    const int64_t lib = row / a.rows_per_lib;
    a.pnv[pos] = min(a.n_valid[lib * a.C + a.idx[pair]], a.page_rows);
    a.qinv[pos] = 1.f / s;
  }
}

// ----------------------------------------------------------------------------------------------------- cluster PTX
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
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
  unsigned char* p;       // [8 blocks][RS_PBLK]
  unsigned char* stages;  // [RS_STAGES][RS_STAGE]
  float* smax;            // [2][2 * cs][MT]: by the parity of the unit (a CTA without scores may lag a unit behind)
  float* ssum;            // [2][2 * cs][MT]
  uint64_t *full, *empty, *s_full, *s_empty, *p_full, *o_full, *o_empty, *stat, *sums;
  uint32_t* tmem;
  volatile int* abort_flag;
};
constexpr size_t RS_SMEM = 1024 + 8 * RS_PBLK + (size_t)RS_STAGES * RS_STAGE + 2 * 4 * RS_MAX_CS * RS_AROWS * 4 +
                           (2 * RS_STAGES + 2 * RS_ACC + 5) * 8 + 16;

__device__ __forceinline__ RsSmem rs_smem(unsigned char* base) {
  RsSmem s;
  s.p = base;
  s.stages = base + 8 * RS_PBLK;
  s.smax = reinterpret_cast<float*>(s.stages + RS_STAGES * RS_STAGE);
  s.ssum = s.smax + 4 * RS_MAX_CS * RS_AROWS;
  s.full = reinterpret_cast<uint64_t*>(s.ssum + 4 * RS_MAX_CS * RS_AROWS);
  s.empty = s.full + RS_STAGES;
  s.s_full = s.empty + RS_STAGES;
  s.s_empty = s.s_full + RS_ACC;
  s.p_full = s.s_empty + RS_ACC;
  s.o_full = s.p_full + 1;
  s.o_empty = s.o_full + 1;
  s.stat = s.o_empty + 1;
  s.sums = s.stat + 1;
  s.tmem = reinterpret_cast<uint32_t*>(s.sums + 1);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem + 1);
  return s;
}

template <typename T, int TERMS>
__global__ void __launch_bounds__(RS_THREADS, 1)
    shared_read_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const SharedArgs a) {
  constexpr int MT = RS_AROWS / TERMS;              // pairs per tile
  constexpr int FMT = std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16;
  constexpr int QUARTERS = RS_AROWS / 32;           // TMEM lane quarters that carry data
  constexpr int CQ = QUARTERS / TERMS;              // quarters of the hi terms: the warps that do the softmax
  constexpr int CW = 2 * CQ, AW = 2 * QUARTERS;     // their warps (two column halves each); warps that read TMEM
  extern __shared__ unsigned char rs_smem_raw[];
  const RsSmem s = rs_smem(reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(rs_smem_raw) + 1023) &
                                                            ~uintptr_t(1023)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = a.cs, ns = a.ns;
  const int rank = (int)cluster_rank();
  const int cluster = blockIdx.x / cs, n_clusters = gridDim.x / cs;
  const int nkb = (a.d_s + 63) / 64;
  const int kpc = TERMS == 2 ? RS_CHUNK : nkb;                    // k-blocks per score accumulator
  const int x0 = rank * a.slab;                                   // this CTA's columns of d_s
  const int my_boxes = max(0, min(a.slab, a.d_s - x0) + 63) / 64;  // in boxes of 64
  const uint32_t blk_bytes = (uint32_t)(ns / 64) * RS_PBLK;       // this CTA's share of P

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    for (int i = 0; i < RS_STAGES; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < RS_ACC; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_empty[i], AW);
    }
    mbar_init(s.p_full, 1);
    mbar_init(s.o_full, 1);
    mbar_init(s.o_empty, AW);
    mbar_init(s.stat, cs * CW);
    mbar_init(s.sums, cs * CW);
    *s.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tc_alloc(s.tmem, 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // every CTA's barriers exist before another CTA arrives on them
  tc_fence_after();
  const uint32_t taddr = *s.tmem;
  pdl_wait();
  const int n_units = *a.n_tiles * a.segs;

  if (warp == 0) {
    // --------------------------------------------------------------------------------------------- producer
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      auto stage = [&](uint32_t bytes) -> unsigned char* {
        const uint32_t st = it % RS_STAGES, use = it / RS_STAGES;
        if (use > 0 && (!mbar_wait_bounded(&s.empty[st], (use - 1) & 1) || *s.abort_flag)) {
          *s.abort_flag = 1;
          ok = false;
          return nullptr;
        }
        mbar_arrive_expect_tx(&s.full[st], bytes);
        ++it;
        return s.stages + st * RS_STAGE;
      };
      for (int u = cluster; u < n_units && ok; u += n_clusters) {
        const SharedTile t = a.tiles[u / a.segs];
        const int seg0 = (u % a.segs) * a.seg_rows;
        const int nv = min(t.nv - seg0, a.seg_rows);
        if (nv <= 0) continue;
        const int y0 = t.page * a.page_rows + seg0;
        if (rank * ns < nv) {
          for (int kb = 0; kb < nkb && ok; ++kb) {
            unsigned char* st = stage((uint32_t)(RS_AROWS * 128 + ns * 128));
            if (!st) break;
            uint64_t* bar = &s.full[(it - 1) % RS_STAGES];
#pragma unroll
            for (int x = 0; x < TERMS; ++x)
              tma_load_2d(st + x * MT * 128, &map_q, kb * 64, x * a.n_pairs + t.start, bar);
            tma_load_2d(st + RS_AROWS * 128, &map_k, kb * 64, y0 + rank * ns, bar);
          }
        }
        for (int b = 0; b < (nv + 63) / 64 && ok; ++b)
          for (int h = 0; h < my_boxes && ok; h += 4) {
            const int n = min(4, my_boxes - h);
            unsigned char* st = stage((uint32_t)n * 64 * 128);
            if (!st) break;
            for (int i = 0; i < n; ++i)
              tma_load_2d(st + i * 64 * 128, &map_v, x0 + (h + i) * 64, y0 + b * 64, &s.full[(it - 1) % RS_STAGES]);
          }
      }
      // the copies in flight end before the CTA's shared memory goes away
      const uint32_t n_last = it < RS_STAGES ? it : RS_STAGES;
      for (uint32_t i = 0; i < n_last; ++i) {
        const uint32_t last = it - 1 - i;
        mbar_wait_bounded(&s.full[last % RS_STAGES], (last / RS_STAGES) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // --------------------------------------------------------------------------------------------- MMA issuer
    uint32_t it = 0, unit = 0, acc = 0;
    bool ok = true;
    auto wait_full = [&]() -> int {  // the next stage, or -1
      const uint32_t st = it % RS_STAGES;
      if (!mbar_wait_bounded(&s.full[st], (it / RS_STAGES) & 1) || *s.abort_flag) {
        *s.abort_flag = 1;
        ok = false;
        return -1;
      }
      ++it;
      tc_fence_after();
      return (int)st;
    };
    const uint32_t id_s = umma_idesc(FMT, FMT, 128, ns);
    for (int u = cluster; u < n_units && ok; u += n_clusters) {
      const SharedTile t = a.tiles[u / a.segs];
      const int nv = min(t.nv - (u % a.segs) * a.seg_rows, a.seg_rows);
      if (nv <= 0) continue;
      if (unit > 0 && (!mbar_wait_bounded(s.o_empty, (unit - 1) & 1) || *s.abort_flag)) {
        *s.abort_flag = 1;
        break;
      }
      tc_fence_after();
      if (rank * ns < nv) {
        for (int kb = 0; kb < nkb; ++kb) {
          const int in = kb % kpc;
          const uint32_t buf = acc % RS_ACC, use = acc / RS_ACC;
          if (in == 0 && use > 0) {
            if (!mbar_wait_bounded(&s.s_empty[buf], (use - 1) & 1) || *s.abort_flag) {
              *s.abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
          }
          const int st = wait_full();
          if (st < 0) break;
          const bool last = in == kpc - 1 || kb == nkb - 1;
          if (lane == 0) {
            const uint32_t sa = smem_u32(s.stages + st * RS_STAGE), sb = sa + RS_AROWS * 128;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc_mma<0>(taddr + buf * (uint32_t)ns, umma_desc_k_sw128(sa + ks * 32), umma_desc_k_sw128(sb + ks * 32),
                        id_s, in > 0 || ks > 0);
            tc_commit(&s.empty[st]);
            if (last) tc_commit(&s.s_full[buf]);
          }
          acc += last;
          __syncwarp();
        }
        if (!ok) break;
      }
      // every CTA's block of P is here (and this CTA's softmax warps have read the scores)
      if (!mbar_wait_cluster(s.p_full, unit & 1) || *s.abort_flag) {
        *s.abort_flag = 1;
        break;
      }
      tc_fence_after();
      for (int b = 0; b < (nv + 63) / 64 && ok; ++b) {
        const int left = nv - b * 64, steps = min(4, (left + 15) / 16);
        for (int h = 0; h < my_boxes; h += 4) {
          const int n = min(4, my_boxes - h);
          const int st = wait_full();
          if (st < 0) break;
          unsigned char* base = s.stages + st * RS_STAGE;
          if (left < steps * 16) {  // rows of V behind the last valid slot: zeros
            for (int i = lane; i < (steps * 16 - left) * n * 8; i += 32) {
              const int r = left + i / (n * 8), c = i % (n * 8);
              *reinterpret_cast<uint4*>(base + (c >> 3) * 64 * 128 + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) {
            const uint32_t sp = smem_u32(s.p + b * RS_PBLK), sv = smem_u32(base);
            const uint32_t id = umma_idesc(FMT, FMT, 128, n * 64, 1);
            for (int ks = 0; ks < steps; ++ks)
              tc_mma<0>(taddr + (uint32_t)h * 64, umma_desc_k_sw128(sp + ks * 32),
                        umma_desc_mn_sw128(sv + ks * 2048, 64 * 128), id, b > 0 || ks > 0);
            tc_commit(&s.empty[st]);
          }
          __syncwarp();
        }
      }
      if (!ok) break;
      if (lane == 0) tc_commit(s.o_full);
      __syncwarp();
      ++unit;
    }
  } else {
    // --------------------------------------------------------------------------------------------- softmax, epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    if (quarter < QUARTERS) {
      const int term = quarter / CQ;                  // 0: hi rows, which do the softmax
      const int row = (quarter % CQ) * 32 + lane;     // pair of the tile
      const uint32_t tl = taddr + ((uint32_t)(quarter * 32) << 16);
      const int hw = ns / 2;                          // score columns of this warp
      // scratch of the lo -> hi hand-over: the block of P that belongs to another CTA (no copy reads it, and none
      // arrives before this CTA's maxima of the unit are out): [columns][rows of a pair of warps]
      float* xch = reinterpret_cast<float*>(s.p + (size_t)((rank + 1 + half) % cs) * blk_bytes) +
                   (quarter % CQ) * 32 * ns;
      uint32_t unit = 0, acc = 0;
      // A wait that runs out sets the abort flag; from then on nothing is waited for, and the warps run through their
      // units on whatever is there, so that the named barriers they share stay matched.
      auto done = [&](bool arrived) {
        if (!arrived) *s.abort_flag = 1;
      };
      for (int u = cluster; u < n_units; u += n_clusters) {
        const SharedTile t = a.tiles[u / a.segs];
        const int seg = u % a.segs, seg0 = seg * a.seg_rows;
        const int nv = min(t.nv - seg0, a.seg_rows);
        if (nv <= 0) continue;
        const bool mine = rank * ns < nv;
        float* smax = s.smax + (unit & 1) * 2 * cs * MT;
        float* ssum = s.ssum + (unit & 1) * 2 * cs * MT;
        const bool live = row < t.count;
        const int pos = t.start + (live ? row : 0);
        const int pnv = live ? a.pnv[pos] - seg0 : 0;            // the pair's valid slots in this segment
        const float c = live ? a.qinv[pos] * a.qscale : 0.f;
        const int c0 = rank * ns + half * hw;                    // first slot of this warp's columns
        float v[64];
        float mx = a.softmax ? -CUDART_INF_F : 0.f;
        if (mine) {
          for (int k0 = 0; k0 < nkb; k0 += kpc, ++acc) {
            const uint32_t buf = acc % RS_ACC;
            done(*s.abort_flag || mbar_wait_bounded(&s.s_full[buf], (acc / RS_ACC) & 1));
            tc_fence_after();
            const uint32_t at = tl + buf * (uint32_t)ns + (uint32_t)(half * hw);
            float x[64];
            if (hw == 64) {
              tc_ld64(at, x);
            } else {
              tc_ld32(at, x);
#pragma unroll
              for (int i = 32; i < 64; ++i) x[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 64; ++i) v[i] = k0 == 0 ? x[i] : v[i] + x[i];
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.s_empty[buf]);
          }
          if (TERMS == 2) {
            if (term == 1)
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i < hw) xch[i * 32 + lane] = v[i];
            fence_proxy_async_smem();  // before another CTA's copy may land on the scratch
            tc_fence_before();         // before the read product may overwrite the scores
            named_bar_sync(2 + half * CQ + quarter % CQ, 64);
            if (term == 0)
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i < hw) v[i] += xch[i * 32 + lane];
          }
        }
        if (term == 0) {
          if (mine) {
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              v[i] *= c;
              if (i < hw && c0 + i < pnv) mx = fmaxf(mx, a.softmax ? v[i] : fabsf(v[i]));
            }
          }
          // the rows' maxima to every CTA of the cluster
          for (int r = 0; r < cs; ++r) st_cluster_f32(cluster_map(&smax[(rank * 2 + half) * MT + row], r), mx);
          __syncwarp();
          if (lane < cs) mbar_arrive_cluster(cluster_map(s.stat, lane));
          done(*s.abort_flag || mbar_wait_cluster(s.stat, unit & 1));
          float m = a.softmax ? -CUDART_INF_F : 0.f;
          for (int r = 0; r < 2 * cs; ++r) m = fmaxf(m, smax[r * MT + row]);
          float l = 0.f;
          if (mine) {
            const float lin = a.softmax ? 0.f : f16_range_scale(m);
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              float p = 0.f;
              if (i < hw && c0 + i < pnv)
                p = a.softmax ? RS_P_SCALE * (TERMS == 2 ? exp2f(v[i] - m) : pf_exp2(v[i] - m)) : v[i] * lin;
              l += p;
              v[i] = p;
            }
            // this row's P in 16 bits: block (c0 / 64), 16-byte chunk j of row r at chunk j ^ (r % 8)
            unsigned char* blk = s.p + (size_t)(c0 >> 6) * RS_PBLK;
            const int j0 = (c0 & 63) >> 3;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (j * 8 < hw) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float r0, r1, q0, q1;
                  hi[e] = pack2<T>(v[j * 8 + 2 * e], v[j * 8 + 2 * e + 1], r0, r1);
                  if (TERMS == 2) lo[e] = pack2<T>(v[j * 8 + 2 * e] - r0, v[j * 8 + 2 * e + 1] - r1, q0, q1);
                }
                const int ch = (j0 + j) ^ (row & 7);
                *reinterpret_cast<uint4*>(blk + row * 128 + ch * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (TERMS == 2)
                  *reinterpret_cast<uint4*>(blk + (MT + row) * 128 + ch * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              }
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
          named_bar_sync(1, 32 * CW);
          if (warp == 4 && lane == 0) {  // quarter 0, half 0
            // the other CTAs' blocks are still to come; then this CTA's block to them
            const int n_work = min(cs, (nv + ns - 1) / ns);
            mbar_arrive_expect_tx(s.p_full, (uint32_t)(n_work - (mine ? 1 : 0)) * blk_bytes);
            if (mine && !*s.abort_flag)
              for (int r = 1; r < cs; ++r) {
                const uint32_t to = (uint32_t)((rank + r) % cs);
                unsigned char* src = s.p + (size_t)rank * blk_bytes;
                bulk_s2s(cluster_map(src, to), src, blk_bytes, cluster_map(s.p_full, to));
              }
          }
          for (int r = 0; r < cs; ++r) st_cluster_f32(cluster_map(&ssum[(rank * 2 + half) * MT + row], r), l);
          __syncwarp();
          if (lane < cs) mbar_arrive_cluster(cluster_map(s.sums, lane));
        }
        // ------------------------------------------------------------------------------------- epilogue
        float coef = 0.f;
        if (term == 0) {
          done(*s.abort_flag || mbar_wait_cluster(s.sums, unit & 1));
          float m = a.softmax ? -CUDART_INF_F : 0.f, l = 0.f;
          for (int r = 0; r < 2 * cs; ++r) {
            m = fmaxf(m, smax[r * MT + row]);
            l += ssum[r * MT + row];
          }
          if (a.softmax) coef = l != 0.f ? 1.f / l : 0.f;
          else coef = pnv + seg0 > 0 ? rsqrtf((float)(pnv + seg0)) / f16_range_scale(m) : 0.f;
          if (live && rank == 0 && half == 0) a.ml[(int64_t)pos * a.segs + seg] = make_float2(m, l);
        }
        done(*s.abort_flag || mbar_wait_bounded(s.o_full, unit & 1));
        tc_fence_after();
        const int cols = my_boxes * 64, pass = 32;
        float* dst = a.part + ((int64_t)pos * a.segs + seg) * a.d_s + x0;
        // the two halves of the warps take alternate passes of 32 columns
        for (int q0 = half * pass; q0 < cols; q0 += 2 * pass) {
          float o[32];
          tc_ld32(tl + (uint32_t)q0, o);
          if (TERMS == 2) {
            if (term == 1)
#pragma unroll
              for (int i = 0; i < 32; ++i) xch[i * 32 + lane] = o[i];
            named_bar_sync(2 + half * CQ + quarter % CQ, 64);
            if (term == 0)
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] += xch[i * 32 + lane];
            named_bar_sync(2 + half * CQ + quarter % CQ, 64);
          }
          if (term == 0 && live) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (x0 + q0 + i < a.d_s)
                *reinterpret_cast<float4*>(dst + q0 + i) =
                    make_float4(o[i] * coef, o[i + 1] * coef, o[i + 2] * coef, o[i + 3] * coef);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s.o_empty);
        ++unit;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while another may still write to its shared memory
  tc_fence_after();
  if (warp == 1) tc_dealloc(taddr, 512);
}

// ----------------------------------------------------------------------------------------------------- combine
// r[row] = sum_j wk[row, j] * (the pair's segments, merged by their maxima and sums), in the order of j.
template <typename TO>
__global__ void __launch_bounds__(256) shared_combine_kernel(const SharedArgs a, TO* __restrict__ r) {
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int64_t lib = row / a.rows_per_lib;
  const int x = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (x >= a.d_s) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < a.k; ++j) {
    const int64_t pair = row * a.k + j;
    const int page = a.page[pair];
    if (page < 0) continue;
    const int64_t pos = a.cnt[page] + a.rank[pair];
    const int nv = min(a.n_valid[lib * a.C + a.idx[pair]], a.page_rows);
    const int segs = (nv + a.seg_rows - 1) / a.seg_rows;
    const float w = a.wk[pair];
    const float* p = a.part + pos * a.segs * a.d_s + x;
    float m = -CUDART_INF_F, z = 0.f;
    if (a.softmax && segs > 1) {
      for (int g = 0; g < segs; ++g) m = fmaxf(m, a.ml[pos * a.segs + g].x);
      for (int g = 0; g < segs; ++g) {
        const float2 ml = a.ml[pos * a.segs + g];
        z += exp2f(ml.x - m) * ml.y;
      }
    }
    for (int g = 0; g < segs; ++g) {
      float f = w;
      if (a.softmax && segs > 1) {
        const float2 ml = a.ml[pos * a.segs + g];
        f *= exp2f(ml.x - m) * ml.y / z;
      }
      const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)g * a.d_s);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
  }
  TO* o = r + row * a.d_s + x;
  o[0] = from_f32<TO>(acc.x);
  o[1] = from_f32<TO>(acc.y);
  o[2] = from_f32<TO>(acc.z);
  o[3] = from_f32<TO>(acc.w);
}

}  // namespace xencb
