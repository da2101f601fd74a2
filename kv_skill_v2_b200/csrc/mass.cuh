// Attention mass: what every slot of a pool receives from a batch of rows,
//
//   mass[p, n] = decay * prior[p, n] + sum over (row t, routed chunk j) with page_of[lib(t), idx[t, j]] = p and
//                n < n_valid[lib(t), idx[t, j]] of wk[t, j] * softmax_n(read_temp * q_t . K_p[n])
//
// the column sums of the weights with which the read (xenc/injector.py:239-245) multiplies the values. The (row, routed
// chunk) pairs are grouped by page in the order of their rows; a tile is one page with up to 128 of its pairs.
//
//   mass_prep    q in 16 bits, a power of two per row (f16's range); CTA 0 counts the pairs of each page and lays out the
//                tiles
//   mass_order   a CTA per page lists its pairs in order, so that sums do not depend on the order of atomics
//   mass_scores  a cluster of ceil(page_rows / 256) CTAs per tile, each with up to 256 of the page's slots:
//                S[pairs, slots] = Q . K^T on the tensor cores (pairs as the 128-row operand), chunk softmax, column sums
//   mass_combine a page's tiles added in order, with the prior
//
// In mass_scores the slots arrive by TMA, the pairs' rows of Q by 16-byte asynchronous copies (128 rows anywhere in the
// batch, so no row is copied in memory for each of its pairs). A pair is a TMEM lane, so the maximum and the sum of its
// softmax stay within a thread; the CTAs of the cluster exchange both through distributed shared memory. A slot's sum over
// 32 pairs is a butterfly over the warp's lanes (31 shuffles for 32 slots).
//
// Precision. Float32 q enters as hi + lo in 16 bits, two products into one accumulator: 22 bits with f16 slots, 16 with
// bf16. A 16-bit q is one product, exact (bf16 q fits f16's 11 bits, but for values 2^-28 below the row's largest). The
// tensor core's accumulator drops bits below its running value, so it runs over MS_CHUNK blocks of 64 columns and is added
// up in float32 registers.
#pragma once

#include <math_constants.h>

#include "read_shared.cuh"

namespace xencb {

constexpr int MS_M = 128;         // pairs of a tile
constexpr int MS_N = 256;         // slots of a CTA at most
constexpr int MS_MAX_CS = 8;      // CTAs per cluster: pages of up to 2048 slots
constexpr int MS_CHUNK = 2;       // blocks of 64 columns per accumulator
constexpr int MS_ATILE = MS_M * 128;
constexpr int MS_BTILE = MS_N * 128;
constexpr int MS_PRODUCERS = 2;   // warps that bring Q
constexpr int MS_EPI = 8;         // softmax warps: 4 TMEM lane quarters x 2 halves of the slots
constexpr int MS_THREADS = 32 * (2 + MS_PRODUCERS + MS_EPI);
constexpr int MS_REGS_LOW = 88, MS_REGS_HIGH = 208;  // registers of a thread of the first four warps, and of the others
constexpr int MS_REGS = 4 * 32 * MS_REGS_LOW + 32 * MS_EPI * MS_REGS_HIGH;
static_assert(2 + MS_PRODUCERS == 4, "the softmax warps begin a group of four");
constexpr int MS_ONE_CTA = 16384;  // pairs that one CTA counts
__host__ __device__ constexpr int ms_stage(int terms) { return terms * MS_ATILE + MS_BTILE; }
// stages of the ring: what the maxima and sums of cs CTAs (two generations, two halves of the slots each) leave
__host__ __device__ constexpr int ms_stages(int terms, int cs) { return (cs <= 4 ? 1 : 0) + (terms == 2 ? 2 : 3); }
__host__ __device__ constexpr size_t ms_smem(int terms, int cs) {
  return 1024 + (size_t)ms_stages(terms, cs) * ms_stage(terms) + (size_t)cs * 4 * MS_M * 8 + 4 * MS_N * 4 + 256;
}

struct __align__(16) MassTile {
  int page, start, count, nv;  // pairs [start, start + count) in grouped order; nv: the most valid slots of the page
};

struct MassArgs {
  const int32_t* page_of;  // [n_lib, C]
  const int32_t* n_valid;  // [n_lib, C]
  const int32_t* idx;      // [R, k]
  const float* wk;         // [R, k]
  int64_t n_rows, rows_per_lib, n_lib;
  int k, C, n_pages, page_rows, d_s, n_pairs;
  // plan
  int* cnt;       // [n_pages]: pairs per page
  int* nvmax;     // [n_pages]
  int* start;     // [n_pages]: the page's first place
  int* tile0;     // [n_pages]: its first tile
  int* page;      // [n_pairs]: page of a pair, -1: reads nothing
  int* prow;      // [n_pairs] by place: row of q
  int* pnv;       // [n_pairs] by place: valid slots
  float* pw;      // [n_pairs] by place: weight
  MassTile* tiles;
  int* n_tiles;
  // rows
  float* rinv;    // [R]: 1 / (the row's power of two)
  const void* q16;  // [terms, R, d_s]
  // scores
  int cs, per;    // CTAs per cluster, slots per CTA
  float qscale;   // read_temp * log2(e)
  float* part;    // [tiles, page_rows]
  const float* prior;
  float decay;
  float* mass;
};

__device__ __forceinline__ void ms_count(const MassArgs& a, int64_t first, int64_t step) {
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
      const int nv = a.n_valid[lib * a.C + c];
      if (nv > a.page_rows) flag_error(XENCB_DEV_CLAMPED);
      if (nv <= 0) {
        page = -1;
      } else {
        atomicAdd(&a.cnt[page], 1);
        atomicMax(&a.nvmax[page], min(nv, a.page_rows));
      }
    }
    a.page[i] = page;
  }
}

__global__ void __launch_bounds__(256) mass_count_kernel(const MassArgs a) {
  ms_count(a, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// First places and tiles of the pages, by one CTA of 1024 threads.
__device__ __forceinline__ void ms_scan(const MassArgs& a) {
  __shared__ int sh[32];
  const int per = (a.n_pages + 1023) / 1024;
  const int p0 = min(a.n_pages, (int)threadIdx.x * per), p1 = min(a.n_pages, p0 + per);
  int pos = 0, tiles = 0;
  for (int p = p0; p < p1; ++p) {
    pos += a.cnt[p];
    tiles += (a.cnt[p] + MS_M - 1) / MS_M;
  }
  int all;
  int at = pg_scan(pos, sh, &all);
  int tile = pg_scan(tiles, sh, &all);
  if (threadIdx.x == 0) *a.n_tiles = all;
  for (int p = p0; p < p1; ++p) {
    const int c = a.cnt[p];
    a.start[p] = at;
    a.tile0[p] = tile;
    for (int s = 0; s < c; s += MS_M) a.tiles[tile++] = MassTile{p, at + s, min(MS_M, c - s), a.nvmax[p]};
    at += c;
  }
}

// CTA 0: the plan (counted: the counts are there already). The others: four rows of q each, 256 threads a row.
constexpr int MS_PREP_THREADS = 1024;
template <typename TQ, typename T, int TERMS>
__global__ void __launch_bounds__(MS_PREP_THREADS) mass_prep_kernel(const MassArgs a, const TQ* __restrict__ q,
                                                                    T* __restrict__ out, int counted) {
  __shared__ float red[32];
  pdl_trigger();
  if (blockIdx.x == 0) {
    if (!counted) {
      for (int p = threadIdx.x; p < a.n_pages; p += MS_PREP_THREADS) {
        a.cnt[p] = 0;
        a.nvmax[p] = 0;
      }
      __syncthreads();
      ms_count(a, threadIdx.x, MS_PREP_THREADS);
      __syncthreads();
    }
    ms_scan(a);
    return;
  }
  const int grp = threadIdx.x >> 8, t = threadIdx.x & 255;
  const int64_t row = ((int64_t)blockIdx.x - 1) * 4 + grp;
  const bool in = row < a.n_rows;
  const TQ* src = q + row * a.d_s;
  float s = 1.f;
  if (std::is_same<T, __half>::value) {  // f16's range: the row's largest value to [2^14, 2^15)
    float mx = 0.f;
    if (in)
      for (int i = t * 8; i < a.d_s; i += 256 * 8) {
        float v[8];
        load8_f32<TQ>(src + i, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[e]));
      }
    mx = warp_max(mx);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = red[grp * 8];
#pragma unroll
    for (int w = 1; w < 8; ++w) mx = fmaxf(mx, red[grp * 8 + w]);
    s = f16_range_scale(mx);
  }
  if (!in) return;
  if (t == 0) a.rinv[row] = 1.f / s;
  for (int i = t * 8; i < a.d_s; i += 256 * 8) {
    float v[8];
    load8_f32<TQ>(src + i, v);
    alignas(16) T hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = from_f32<T>(v[e] * s);
      if (TERMS == 2) lo[e] = from_f32<T>(v[e] * s - to_f32(hi[e]));
    }
    *reinterpret_cast<uint4*>(out + row * a.d_s + i) = *reinterpret_cast<const uint4*>(hi);
    if (TERMS == 2)
      *reinterpret_cast<uint4*>(out + (a.n_rows + row) * a.d_s + i) = *reinterpret_cast<const uint4*>(lo);
  }
}

// One CTA per page: its pairs in the order of their rows.
constexpr int MS_ORDER_THREADS = 256;
__global__ void __launch_bounds__(MS_ORDER_THREADS) mass_order_kernel(const MassArgs a) {
  __shared__ int sh[MS_ORDER_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int p = blockIdx.x, n = a.cnt[p], start = a.start[p];
  if (n == 0) return;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int found = 0;
  for (int64_t i0 = 0; i0 < a.n_pairs && found < n; i0 += MS_ORDER_THREADS * 4) {
    const int64_t i = i0 + threadIdx.x * 4;
    int hit[4], c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hit[e] = i + e < a.n_pairs && a.page[i + e] == p;
      c += hit[e];
    }
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) sh[wid] = incl;
    __syncthreads();
    int at = found + incl - c;
#pragma unroll
    for (int w = 0; w < MS_ORDER_THREADS / 32; ++w) {
      at += w < wid ? sh[w] : 0;
      found += sh[w];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (hit[e]) {
        const int64_t row = (i + e) / a.k;
        const int place = start + at++;
        a.prow[place] = (int)row;
        a.pnv[place] = min(a.n_valid[row / a.rows_per_lib * a.C + a.idx[i + e]], a.page_rows);
        a.pw[place] = a.wk[i + e];
      }
  }
}

// ----------------------------------------------------------------------------------------------------- scores
// 16 bytes from global to shared memory, and the arrival on `bar` of everything this thread has asked for so far.
__device__ __forceinline__ void ms_copy16(uint32_t dst, const void* src, uint32_t bytes) {  // (zeros behind `bytes`)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ms_copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

struct MsSmem {
  unsigned char* stages;
  float* stat;   // [2][2 cs][128][2]: by the parity of the tile, maximum and sum of each pair's half of a CTA's slots
  float* cols;   // [4][256]: column sums of the lane quarters
  uint64_t *full, *empty, *s_full, *s_empty, *st;
  uint32_t* tmem;
  volatile int* abort_flag;
};

template <typename T, int TERMS>
__global__ void __launch_bounds__(MS_THREADS, 1)
    mass_scores_kernel(const __grid_constant__ CUtensorMap map_k, const MassArgs a) {
  constexpr int FMT = std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16;
  constexpr int STAGE = ms_stage(TERMS);
  extern __shared__ unsigned char ms_smem_raw[];
  const int cs = a.cs, n_st = ms_stages(TERMS, cs);
  MsSmem s;
  s.stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ms_smem_raw) + 1023) & ~uintptr_t(1023));
  s.stat = reinterpret_cast<float*>(s.stages + n_st * STAGE);
  s.cols = s.stat + cs * 4 * MS_M * 2;
  s.full = reinterpret_cast<uint64_t*>(s.cols + 4 * MS_N);
  s.empty = s.full + 4;
  s.s_full = s.empty + 4;
  s.s_empty = s.s_full + 2;
  s.st = s.s_empty + 2;
  s.tmem = reinterpret_cast<uint32_t*>(s.st + 2);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int cluster = blockIdx.x / cs, n_clusters = gridDim.x / cs;
  const int nkb = (a.d_s + 63) / 64, n_chunk = (nkb + MS_CHUNK - 1) / MS_CHUNK;
  const int seg0 = rank * a.per;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_k);
    for (int i = 0; i < n_st; ++i) {
      mbar_init(&s.full[i], 1 + 32 * MS_PRODUCERS);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_empty[i], MS_EPI);
    }
    // the statistics of even and odd tiles: one arrival and the bytes of cs * 2 * 128 pairs. (A CTA may be a tile ahead of
    // another, whose barrier for the tile before still waits for a third.)
    mbar_init(&s.st[0], 1);
    mbar_init(&s.st[1], 1);
    *s.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tc_alloc(s.tmem, 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t taddr = *s.tmem;
  pdl_wait();
  const int n_tiles = *a.n_tiles;
  auto done = [&](bool arrived) {
    if (!arrived) *s.abort_flag = 1;
    __syncwarp();
  };

  // The softmax keeps 128 sums a thread: the other warps give registers up (their sum stays below the launch's).
  if (warp < 4) {
    regs_dec<MS_REGS_LOW>();
    if (warp == 0) {
      // --------------------------------------------------------------------------------------------- slots
      if (elect_one()) {
        RsRing ring{0, 0};
        uint32_t used = 0;
        bool ok = true;
        for (int t = cluster; t < n_tiles && ok; t += n_clusters) {
          const MassTile tile = a.tiles[t];
          if (seg0 >= tile.nv) continue;
          const int y = tile.page * a.page_rows + seg0;
          for (int kb = 0; kb < nkb; ++kb) {
            if (used >= (uint32_t)n_st && !(ok = mbar_wait_spin(&s.empty[ring.st], ring.phase ^ 1))) break;
            mbar_arrive_expect_tx(&s.full[ring.st], (uint32_t)a.per * 128);
            tma_load_2d(s.stages + ring.st * STAGE + TERMS * MS_ATILE, &map_k, kb * 64, y, &s.full[ring.st]);
            ring.next(n_st);
            ++used;
          }
        }
        if (!ok) {  // the copies in flight end before the CTA's shared memory goes away
          *s.abort_flag = 1;
          for (uint32_t i = min(used, (uint32_t)n_st); i > 0; --i) {
            ring.back(n_st);
            mbar_wait_bounded(&s.full[ring.st], ring.phase);
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // --------------------------------------------------------------------------------------------- MMA issuer
      if (elect_one()) {
        RsRing ring{0, 0};
        uint32_t acc = 0;
        bool ok = true;
        const uint32_t idesc = umma_idesc(FMT, FMT, MS_M, a.per);
        for (int t = cluster; t < n_tiles && ok; t += n_clusters) {
          if (seg0 >= a.tiles[t].nv) continue;
          for (int k0 = 0; k0 < nkb && ok; k0 += MS_CHUNK, ++acc) {
            const uint32_t buf = acc & 1, use = acc >> 1;
            if (use > 0 && !(ok = mbar_wait_spin(&s.s_empty[buf], (use - 1) & 1))) break;
            tc_fence_after();
            const int k1 = min(nkb, k0 + MS_CHUNK);
            for (int kb = k0; kb < k1; ++kb) {
              if (!(ok = mbar_wait_spin(&s.full[ring.st], ring.phase))) break;
              fence_proxy_async_smem();  // Q was written by this CTA's threads
              tc_fence_after();
              const uint32_t st = smem_u32(s.stages + ring.st * STAGE), bk = st + TERMS * MS_ATILE;
  #pragma unroll
              for (int ks = 0; ks < 4; ++ks)
  #pragma unroll
                for (int x = 0; x < TERMS; ++x)
                  tc_mma<0>(taddr + buf * MS_N, umma_desc_k_sw128(st + x * MS_ATILE + ks * 32),
                            umma_desc_k_sw128(bk + ks * 32), idesc, kb > k0 || ks > 0 || x > 0);
              tc_commit(&s.empty[ring.st]);
              ring.next(n_st);
            }
            if (ok) tc_commit(&s.s_full[buf]);
          }
        }
        if (!ok) *s.abort_flag = 1;
      }
      __syncwarp();
    } else {
      // --------------------------------------------------------------------------------------------- rows of Q
      // Eight lanes a row (16 bytes each: chunk j of row r at chunk j ^ (r % 8)), 4 MS_PRODUCERS rows at a time.
      constexpr int STEP = 4 * MS_PRODUCERS, PASSES = MS_M / STEP;
      const int t0 = threadIdx.x - 64;
      const int sub = t0 >> 3, ch = t0 & 7;
      const char* q = static_cast<const char*>(a.q16);
      const int64_t row_bytes = (int64_t)a.d_s * 2, lo = a.n_rows * row_bytes;
      RsRing ring{0, 0};
      uint32_t used = 0;
      bool ok = true;
      for (int t = cluster; t < n_tiles && ok; t += n_clusters) {
        const MassTile tile = a.tiles[t];
        if (seg0 >= tile.nv) continue;
        int rows[PASSES];
  #pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int r = i * STEP + sub;
          rows[i] = r < tile.count ? a.prow[tile.start + r] : -1;
        }
        for (int kb = 0; kb < nkb; ++kb) {
          if (used >= (uint32_t)n_st) {
            ok = mbar_wait_spin(&s.empty[ring.st], ring.phase ^ 1);
            if (!ok) break;
          }
          const uint32_t st = smem_u32(s.stages + ring.st * STAGE);
          const int col = kb * 64 + ch * 8;
          const bool in = col < a.d_s;
  #pragma unroll
          for (int i = 0; i < PASSES; ++i) {
            if (i * STEP >= tile.count) break;
            const int r = i * STEP + sub;
            if (rows[i] >= 0) {  // columns behind d_s: zeros, as the slots' are
              const char* src = q + rows[i] * row_bytes + (in ? col * 2 : 0);
              const uint32_t dst = st + r * 128 + ((ch ^ (r & 7)) << 4);
              ms_copy16(dst, src, in ? 16 : 0);
              if (TERMS == 2) ms_copy16(dst + MS_ATILE, src + lo, in ? 16 : 0);
            }
          }
          ms_copies_arrive(&s.full[ring.st]);
          ring.next(n_st);
          ++used;
        }
      }
      if (!ok) *s.abort_flag = 1;
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
  } else {
    // --------------------------------------------------------------------------------------------- softmax
    regs_inc<MS_REGS_HIGH>();
    const int quarter = warp & 3, half = (warp - 2 - MS_PRODUCERS) >> 2;
    const int r = quarter * 32 + lane;               // pair of the tile = TMEM lane
    const uint32_t tl = taddr + ((uint32_t)(quarter * 32) << 16) + half * 128;
    const int n0 = seg0 + half * 128;                // first slot of this warp
    const int width = max(0, min(128, a.per - half * 128));
    uint32_t acc = 0, gen = 0;
    for (int t = cluster; t < n_tiles; t += n_clusters, ++gen) {
      const MassTile tile = a.tiles[t];
      const bool here = r < tile.count, any = quarter * 32 < tile.count;
      int nv = 0;
      float w = 0.f, c = 0.f;
      if (here) {
        const int place = tile.start + r;
        nv = min(width, a.pnv[place] - n0);
        w = a.pw[place];
        c = a.rinv[a.prow[place]] * a.qscale;
      }
      float v[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) v[i] = 0.f;
      if (seg0 < tile.nv) {
        for (int k = 0; k < n_chunk; ++k, ++acc) {
          const uint32_t buf = acc & 1;
          done(*s.abort_flag || mbar_wait_spin(&s.s_full[buf], (acc >> 1) & 1));
          tc_fence_after();
          if (any && width > 0) {
#pragma unroll
            for (int g = 0; g < 128; g += 32) {
              float x[32];
              tc_ld32(tl + buf * MS_N + g, x);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[g + i] += x[i];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.s_empty[buf]);
          __syncwarp();
        }
      }
      // e^(score - max) of this half, its maximum and sum
      float m = -CUDART_INF_F, l = 0.f;
#pragma unroll
      for (int i = 0; i < 128; ++i) {
        v[i] *= c;
        if (i < nv) m = fmaxf(m, v[i]);
      }
#pragma unroll
      for (int i = 0; i < 128; ++i) {
        v[i] = i < nv ? pf_exp2(v[i] - m) : 0.f;
        l += v[i];
      }
      float* stat = s.stat + (size_t)(gen & 1) * cs * 2 * MS_M * 2;
      if (threadIdx.x == 32 * (2 + MS_PRODUCERS)) mbar_arrive_expect_tx(&s.st[gen & 1], (uint32_t)cs * 2 * MS_M * 8);
      {
        float* mine = stat + ((rank * 2 + half) * MS_M + r) * 2;
        for (int to = 0; to < cs; ++to) {
          const uint32_t bar = cluster_map(&s.st[gen & 1], to), dst = cluster_map(mine, to);
          st_async_f32(dst, m, bar);
          st_async_f32(dst + 4, l, bar);
        }
      }
      done(*s.abort_flag || mbar_wait_cluster(&s.st[gen & 1], (gen >> 1) & 1));
      float M = -CUDART_INF_F, L = 0.f;
      for (int e = 0; e < 2 * cs; ++e) M = fmaxf(M, stat[(e * MS_M + r) * 2]);
      for (int e = 0; e < 2 * cs; ++e) {
        const float me = stat[(e * MS_M + r) * 2], le = stat[(e * MS_M + r) * 2 + 1];
        if (me != -CUDART_INF_F) L += le * exp2f(me - M);
      }
      const float f = here && nv > 0 ? w / L * exp2f(m - M) : 0.f;
      // column sums over the warp's pairs, then over the lane quarters
#pragma unroll
      for (int g = 0; g < 128; g += 32) {
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = g + i < nv ? v[g + i] * f : 0.f;
        const float sum = any ? rs_reduce<32>(x, lane, [](float p, float q) { return p + q; }) : 0.f;
        s.cols[quarter * MS_N + half * 128 + g + lane] = sum;
      }
      named_bar_sync(1, 32 * MS_EPI);
      const int col = (int)threadIdx.x - 32 * (2 + MS_PRODUCERS);
      if (col < a.per && seg0 + col < a.page_rows) {
        float sum = s.cols[col];
#pragma unroll
        for (int g = 1; g < 4; ++g) sum += s.cols[g * MS_N + col];
        a.part[(int64_t)t * a.page_rows + seg0 + col] = sum;
      }
      named_bar_sync(1, 32 * MS_EPI);
    }
  }
  __syncwarp();
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while another may still write to its shared memory
  tc_fence_after();
  if (warp == 1) tc_dealloc(taddr, 512);
}

// mass = decay * prior + a page's tiles in order. Grid (n_pages, ceil(page_rows / 256)).
__global__ void __launch_bounds__(256) mass_combine_kernel(const MassArgs a) {
  pdl_wait();
  const int p = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x;
  if (n >= a.page_rows) return;
  const int64_t at = (int64_t)p * a.page_rows + n;
  float v = a.prior ? a.decay * a.prior[at] : 0.f;
  const int tiles = (a.cnt[p] + MS_M - 1) / MS_M;
  const float* part = a.part + (int64_t)a.tile0[p] * a.page_rows + n;
  for (int t = 0; t < tiles; ++t) v += part[(int64_t)t * a.page_rows];
  a.mass[at] = v;
}

}  // namespace xencb
