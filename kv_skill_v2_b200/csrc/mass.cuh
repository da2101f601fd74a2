// Attention mass: what every slot of a pool receives from a batch of rows,
//
//   mass[p, n] = decay * prior[p, n] + sum over (row t, routed chunk j) with page_of[lib(t), idx[t, j]] = p and
//                n < n_valid[lib(t), idx[t, j]] of wk[t, j] * softmax_n(read_temp * q_t . K_p[n])
//
// the column sums of the weights with which the read (xenc/injector.py:239-245) multiplies the values. The (row, routed
// chunk) pairs are grouped by page in the order of their rows; a tile is one page with up to 128 of its pairs.
//
//   mass_plan    counts the pairs of each page and lays out the tiles. Calls of up to MS_DIRECT pairs do without: every page
//                has room for all of them
//   mass_rows    a CTA per page lists its pairs in order, so that sums do not depend on the order of atomics; a CTA per row
//                brings q into 16 bits, a power of two per row (f16's range)
//   mass_scores  a cluster of ceil(page_rows / 256) CTAs per tile, each with up to 256 of the page's slots:
//                S[pairs, slots] = Q . K^T on the tensor cores (pairs as the 128-row operand), chunk softmax, column sums
//                (all a page's tiles, in their order and with the prior, are added up by the CTA that finishes its part of
//                the page last; pages that nothing reads are mass_rows')
//
// In mass_scores the slots arrive by TMA, the pairs' rows of Q by 16-byte asynchronous copies (128 rows anywhere in the
// batch, so no row is copied in memory for each of its pairs). A pair is a TMEM lane, so the maximum and the sum of its
// softmax stay within a thread; the CTAs of the cluster exchange both through distributed shared memory. A slot's sum over
// 32 pairs is a butterfly over the warp's lanes (31 shuffles for 32 slots).
//
// Precision. Float32 q enters as hi + lo in 16 bits, two products into one accumulator: 22 bits with f16 slots, 16 with
// bf16. There a pair's weights come out 12 * 2^-17 / sqrt(d_s) and so off, which a sum over many pairs averages out (measured,
// in norm: 3.5e-6 sqrt(64 / d_s) / sqrt(pairs a page)) and few do not: calls with pairs * d_s < MS_THREE * pages, which wait
// for latency anyway, take hi + mid + lo, 24 bits (64 columns, 6 pairs a page: 1.4e-6 -> 1.1e-7). A 16-bit q is exact: one
// product, two for an f16 q with bf16 slots (bf16 q fits f16's 11 bits, but for values 2^-28 below the row's largest). The
// tensor core's accumulator drops bits below its running value, so it runs over MS_CHUNK or MS_CHUNK_FEW blocks of 64 columns
// and is added up in float32 registers.
//
// What bounds it. Few pairs a page: HBM, one pass over the slots (64 rows on 64 pages of 512 x 2048: 37 us a launch, 3.6
// TB/s; 1024 pages with few pairs each run at 5.6 TB/s). Full tiles: 128 pairs x 512 slots x 2048 columns take 22.9 us of
// products (165 cycles per M 128, N 256, K 16) on a cluster of two, hi and lo; the softmax adds 5 us a tile (softmax 3.2k
// cycles, exchange 1.9k, column sums 3.9k), which the next tile's products do not cover: 4096 float32 rows with 4 of 64
// pages each take 95 us, 0.44 of the rate of the products alone (a 16-bit q 70). Listing the pairs is pages x pairs, as every
// page's CTA reads every pair's page: 15 us of the rows' launch there, 136 with all 64 pages a row (scores 900), 1000 with
// 16384 rows, 128 of 1024 pages each (scores 7300).
#pragma once

#include <math_constants.h>

#include "read_shared.cuh"

namespace xencb {

constexpr int MS_M = 128;         // pairs of a tile
constexpr int MS_N = 256;         // slots of a CTA at most
constexpr int MS_MAX_CLUSTERS = 256;  // of a launch
constexpr int MS_MAX_CS = 8;      // CTAs per cluster: pages of up to 2048 slots
constexpr int MS_CHUNK = 4;       // blocks of 64 columns per accumulator
constexpr int MS_CHUNK_FEW = 2;   // of calls of few pairs, whose errors no sum averages out (64 rows, top-4: 5.6e-7 -> 3.3e-7);
                                  // it costs them nothing, prompts 3 % for the same error
constexpr int MS_THREE = 4096;    // (3.5e-6 / 8 = 4.4e-7 off from there on)
constexpr int MS_ATILE = MS_M * 128;
constexpr int MS_BTILE = MS_N * 128;
constexpr int MS_PRODUCERS = 4;   // warps that bring Q
constexpr int MS_EPI = 8;         // softmax warps: 4 TMEM lane quarters x 2 halves of the slots
constexpr int MS_LOW = 8;         // warps before the softmax: 0 slots, 1 MMA, 4 .. 7 Q
constexpr int MS_THREADS = 32 * (MS_LOW + MS_EPI);
constexpr int MS_REGS_LOW = 56, MS_REGS_HIGH = 200;  // registers of a thread of these warps, and of the others
constexpr int MS_REGS = 32 * (MS_LOW * MS_REGS_LOW + MS_EPI * MS_REGS_HIGH);
constexpr int MS_FEW = 64;        // pairs of a tile whose hi and lo rows fit one 128-row operand
__host__ __device__ constexpr int ms_few(int terms) { return terms == 3 ? 32 : MS_FEW; }  // (or hi, mid and lo rows)
constexpr int MS_ONE_CTA = 2048;  // pairs that one CTA counts
constexpr int MS_DIRECT = 512;    // pairs of a call without a plan
constexpr int MS_XPITCH = 17;     // 16 columns of the lo rows' sums on their way to the hi rows' lanes
__host__ __device__ constexpr int ms_stage(int terms) { return terms * MS_ATILE + MS_BTILE; }
// stages of the ring: what the maxima and sums of cs CTAs (two generations, two halves of the slots each) leave
__host__ __device__ constexpr int ms_stages(int terms, int cs) {
  return terms == 3 ? 2 : (cs <= 4 ? 1 : 0) + (terms == 2 ? 2 : 3);
}
__host__ __device__ constexpr size_t ms_smem(int terms, int cs) {
  return 1024 + (size_t)ms_stages(terms, cs) * ms_stage(terms) + (size_t)cs * 4 * MS_M * 8 + 4 * MS_N * 4 +
         (terms >= 2 ? 2 * MS_FEW * MS_XPITCH * 4 : 0) + 256;
}

struct __align__(16) MassTile {
  int page, start, count, nv;    // pairs [start, start + count) in grouped order; nv: the most valid slots of the page
  int total, base, stride, few;  // tiles of the page: base + j * stride for j < total, the last one `few` if that is not -1
};

struct MassArgs {
  const int32_t* page_of;  // [n_lib, C]
  const int32_t* n_valid;  // [n_lib, C]
  const int32_t* idx;      // [R, k]
  const float* wk;         // [R, k]
  int64_t n_rows;
  int rows_per_lib, k, C, n_pages, page_rows, d_s, n_pairs;
  // plan
  int* cnt;       // [n_pages]: pairs per page
  int* nvmax;     // [n_pages]
  int* start;     // [n_pages]: the page's first place
  int* done;      // [n_pages, cs]: tiles that are finished
  int* page;      // [n_pairs]: page of a pair, -1: reads nothing
  int* prow;      // [n_pairs] by place: row of q
  int* pnv;       // [n_pairs] by place: valid slots
  float* pw;      // [n_pairs] by place: weight
  MassTile* tiles;
  int* n_tiles;
  int direct;     // no plan: page p's pairs from place p * n_pairs on, its j-th tile is tile j * n_pages + p
  int slots;      // of the list of tiles (those without pairs are skipped)
  // rows
  float* rinv;    // [R]: 1 / (the row's power of two)
  const void* q16;  // [terms, R, d_s]: hi, (mid,) lo
  // scores
  int cs, per;    // CTAs per cluster, slots per CTA
  float qscale;   // read_temp * log2(e)
  float* part;    // [tiles, page_rows]
  const float* prior;
  float decay;
  float* mass;
};

// The page that pair i reads and its valid slots; -1: none. Bad tables are flagged where `flag` is set. A weight of NaN, the
// routing of a query that is not finite, reads nothing, as 0 does: the sums are added to call after call.
__device__ __forceinline__ int ms_page(const MassArgs& a, int i, bool flag, int* nv) {
  const int c = a.idx[i];
  if (c < 0 || !(fabsf(a.wk[i]) > 0.f)) return -1;
  const int64_t at = (int64_t)((unsigned)i / (unsigned)a.k / (unsigned)a.rows_per_lib) * a.C + c;
  const int page = c < a.C ? a.page_of[at] : -1;
  if (page < 0 || page >= a.n_pages) {
    if (flag) flag_error(XENCB_DEV_BADPAGE);
    return -1;
  }
  const int n = a.n_valid[at];
  if (flag && n > a.page_rows) flag_error(XENCB_DEV_CLAMPED);
  *nv = min(n, a.page_rows);
  return n > 0 ? page : -1;
}

__device__ __forceinline__ void ms_count(const MassArgs& a, unsigned first, unsigned step) {
  for (unsigned i = first; i < (unsigned)a.n_pairs; i += step) {
    int nv;
    const int page = ms_page(a, i, true, &nv);
    if (page >= 0) {
      atomicAdd(&a.cnt[page], 1);
      atomicMax(&a.nvmax[page], nv);
    }
    a.page[i] = page;
  }
}

constexpr int MS_THREADS_256 = 256;  // of the plan and of the rows
// Exclusive count over the CTA's threads; *total gets the sum. `sh` holds a round's sums of the warps.
__device__ __forceinline__ int ms_scan(int c, int* sh, int* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int incl = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) sh[wid] = incl;
  __syncthreads();
  int before = incl - c, all = 0;
#pragma unroll
  for (int w = 0; w < MS_THREADS_256 / 32; ++w) {
    before += w < wid ? sh[w] : 0;
    all += sh[w];
  }
  *total = all;
  return before;
}

// Counts the pairs; the CTA that ends last lays out places and tiles. The clusters take the tiles in turn (cluster c tiles
// c, c + n_clusters, ...). Those of more than MS_FEW pairs come first; those of few pairs take about half as long: the
// clusters that have one turn less than others get two of them before anybody else gets one, so some turns stay empty.
constexpr int MS_PLAN_THREADS = MS_THREADS_256;
__global__ void __launch_bounds__(MS_PLAN_THREADS) mass_plan_kernel(const MassArgs a, int n_clusters) {
  __shared__ int sh[MS_PLAN_THREADS / 32];
  __shared__ int last;
  pdl_trigger();
  if (gridDim.x == 1) {
    for (int p = threadIdx.x; p < a.n_pages; p += MS_PLAN_THREADS) {
      a.cnt[p] = 0;
      a.nvmax[p] = 0;
    }
    __syncthreads();
  }
  ms_count(a, blockIdx.x * MS_PLAN_THREADS + threadIdx.x, gridDim.x * MS_PLAN_THREADS);
  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&a.nvmax[a.n_pages], 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
  } else {
    __syncthreads();
  }
  const int per = (a.n_pages + MS_PLAN_THREADS - 1) / MS_PLAN_THREADS;
  const int p0 = min(a.n_pages, (int)threadIdx.x * per), p1 = min(a.n_pages, p0 + per);
  int pos = 0, big = 0, few = 0;
  for (int p = p0; p < p1; ++p) {
    const int c = __ldcg(a.cnt + p), left = c % MS_M;
    pos += c;
    big += c / MS_M + (left > MS_FEW);
    few += left > 0 && left <= MS_FEW;
  }
  int all, n_big, n_few;
  int at = ms_scan(pos, sh, &all);
  int tb = ms_scan(big, sh, &n_big);
  int tf = ms_scan(few, sh, &n_few);
  // the j-th tile of few pairs: `gap` clusters have a turn less, and get the first 2 gap of them
  const int taken = n_big % n_clusters, gap = taken ? n_clusters - taken : 0, round = n_big - taken;  // (round: its first turn)
  auto few_at = [&](int j) {
    if (j < gap) return n_big + j;
    if (j < 2 * gap) return round + n_clusters + taken + (j - gap);
    return round + (gap ? 2 * n_clusters : 0) + (j - 2 * gap);
  };
  // (clusters without a hole in the second of these turns leave it empty)
  if (n_few > gap)
    for (int i = threadIdx.x; i < taken; i += MS_PLAN_THREADS) a.tiles[round + n_clusters + i].count = 0;
  if (threadIdx.x == 0) *a.n_tiles = n_few > 0 ? few_at(n_few - 1) + 1 : n_big;
  for (int p = p0; p < p1; ++p) {
    const int c = __ldcg(a.cnt + p), nv = __ldcg(a.nvmax + p);
    a.start[p] = at;
    const int left = c % MS_M, total = (c + MS_M - 1) / MS_M, base = tb;
    const int mine = left > 0 && left <= MS_FEW ? few_at(tf++) : -1;
    for (int s = 0; s < c; s += MS_M) {
      const int n = min(MS_M, c - s);
      a.tiles[mine >= 0 && n < MS_M ? mine : tb++] = MassTile{p, at + s, n, nv, total, base, 1, mine};
    }
    at += c;
  }
}

constexpr int MS_ROWS_THREADS = MS_THREADS_256;
constexpr int MS_ROWS_IDS = 16;  // pairs a thread looks at in one round

// The pairs of page p in the order of their rows.
__device__ __forceinline__ void ms_order(const MassArgs& a, int p) {
  __shared__ int sh[MS_ROWS_THREADS / 32];
  __shared__ int nv_most;
  if (threadIdx.x == 0) nv_most = 0;
  if (threadIdx.x < a.cs) a.done[p * a.cs + threadIdx.x] = 0;
  const int n = a.direct ? a.n_pairs : a.cnt[p];
  const int64_t start = a.direct ? (int64_t)p * a.n_pairs : a.start[p];
  int found = 0;
  const int ids = a.direct ? MS_DIRECT / MS_ROWS_THREADS : MS_ROWS_IDS;  // pairs of a thread in one round
  for (int64_t i0 = 0; i0 < a.n_pairs && found < n; i0 += MS_ROWS_THREADS * ids) {
    const int64_t i = i0 + threadIdx.x * ids;
    uint32_t hit = 0;
    if (a.direct) {
#pragma unroll
      for (int e = 0; e < MS_DIRECT / MS_ROWS_THREADS; ++e) {
        int nv;
        if (i + e < a.n_pairs) hit |= (uint32_t)(ms_page(a, (int)i + e, p == 0, &nv) == p) << e;
      }
    } else {
      int id[MS_ROWS_IDS];
#pragma unroll
      for (int e = 0; e < MS_ROWS_IDS; e += 4) {
        if (i + e + 4 <= a.n_pairs) {
          *reinterpret_cast<int4*>(id + e) = *reinterpret_cast<const int4*>(a.page + i + e);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) id[e + x] = i + e + x < a.n_pairs ? a.page[i + e + x] : -1;
        }
      }
#pragma unroll
      for (int e = 0; e < MS_ROWS_IDS; ++e) hit |= (uint32_t)(id[e] == p) << e;
    }
    int round;
    int64_t place = start + found + ms_scan(__popc(hit), sh, &round);
    found += round;
    for (; hit; hit &= hit - 1, ++place) {
      const unsigned j = (unsigned)i + __ffs(hit) - 1, row = j / (unsigned)a.k;
      const int nv = min(a.n_valid[(int64_t)(row / (unsigned)a.rows_per_lib) * a.C + a.idx[j]], a.page_rows);
      a.prow[place] = (int)row;
      a.pnv[place] = nv;
      a.pw[place] = a.wk[j];
      if (a.direct) atomicMax(&nv_most, nv);
    }
  }
  if (found == 0)
    for (int i = threadIdx.x; i < a.page_rows; i += MS_ROWS_THREADS) {
      const int64_t at = (int64_t)p * a.page_rows + i;
      a.mass[at] = a.prior ? a.decay * a.prior[at] : 0.f;
    }
  if (!a.direct) return;
  __syncthreads();
  const int per = a.slots / a.n_pages, total = (found + MS_M - 1) / MS_M;
  if (threadIdx.x < per) {
    const int s = threadIdx.x * MS_M;
    a.tiles[threadIdx.x * a.n_pages + p] =
        MassTile{p, (int)(start + s), max(0, min(MS_M, found - s)), nv_most, total, p, a.n_pages, -1};
  }
}

// CTAs 0 .. n_pages - 1: a page's pairs; the others: a row of q each.
template <typename TQ, typename T, int TERMS>
__global__ void __launch_bounds__(MS_ROWS_THREADS) mass_rows_kernel(const MassArgs a, const TQ* __restrict__ q,
                                                                    T* __restrict__ out) {
  __shared__ float red[MS_ROWS_THREADS / 32];
  pdl_trigger();
  if ((int)blockIdx.x < a.n_pages) {
    pdl_wait();
    ms_order(a, blockIdx.x);
    return;
  }
  // (No wait: the plan is a plain launch, so whatever wrote q or used this workspace has completed, and it touches neither
  // of the rows' outputs.)
  const int64_t row = (int64_t)blockIdx.x - a.n_pages;
  const TQ* src = q + row * a.d_s;
  constexpr int STEP = MS_ROWS_THREADS * 8, HELD = 2;  // the first HELD pieces stay in registers
  float v[HELD][8];
  float mx = 0.f;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int i = h * STEP + threadIdx.x * 8;
    if (i < a.d_s) {
      load8_f32<TQ>(src + i, v[h]);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(v[h][e]));
    }
  }
  float s = 1.f;
  if (std::is_same<T, __half>::value) {  // f16's range: the row's largest value to [2^14, 2^15)
    for (int i = HELD * STEP + threadIdx.x * 8; i < a.d_s; i += STEP) {
      float w[8];
      load8_f32<TQ>(src + i, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(w[e]));
    }
    mx = warp_max(mx);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
    mx = red[0];
#pragma unroll
    for (int w = 1; w < MS_ROWS_THREADS / 32; ++w) mx = fmaxf(mx, red[w]);
    s = f16_range_scale(mx);
  }
  if (threadIdx.x == 0) a.rinv[row] = 1.f / s;
  auto emit = [&](int i, const float* w) {
    float left[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) left[e] = w[e] * s;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      alignas(16) T x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = from_f32<T>(left[e]);
        left[e] -= to_f32(x[e]);
      }
      *reinterpret_cast<uint4*>(out + (t * a.n_rows + row) * a.d_s + i) = *reinterpret_cast<const uint4*>(x);
    }
  };
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int i = h * STEP + threadIdx.x * 8;
    if (i < a.d_s) emit(i, v[h]);
  }
  for (int i = HELD * STEP + threadIdx.x * 8; i < a.d_s; i += STEP) {
    float w[8];
    load8_f32<TQ>(src + i, w);
    emit(i, w);
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
  float* xch;    // [2][64][MS_XPITCH]: sums of the lo rows of few pairs, or of the mid and the lo rows
  uint64_t *full, *empty, *s_full, *s_empty, *st;
  uint32_t* tmem;
  volatile int *abort_flag, *last;
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
  s.xch = s.cols + 4 * MS_N;
  s.full = reinterpret_cast<uint64_t*>(s.xch + (TERMS >= 2 ? 2 * MS_FEW * MS_XPITCH : 0));
  s.empty = s.full + 4;
  s.s_full = s.empty + 4;
  s.s_empty = s.s_full + 2;
  s.st = s.s_empty + 2;
  s.tmem = reinterpret_cast<uint32_t*>(s.st + 2);
  s.abort_flag = reinterpret_cast<volatile int*>(s.tmem + 1);
  s.last = s.abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int cluster = blockIdx.x / cs, n_clusters = gridDim.x / cs;
  const int nkb = (a.d_s + 63) / 64, chunk = a.direct ? MS_CHUNK_FEW : MS_CHUNK;
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
  const int n_tiles = a.direct ? a.slots : *a.n_tiles;
  auto stacked = [](const MassTile& t) { return TERMS >= 2 && t.count <= ms_few(TERMS); };
  auto done = [&](bool arrived) {
    if (!arrived) *s.abort_flag = 1;
    __syncwarp();
  };

  // The softmax keeps 128 sums a thread: the other warps give registers up (their sum stays below the launch's).
  if (warp < MS_LOW) {
    regs_dec<MS_REGS_LOW>();
    if (warp == 0) {
      // --------------------------------------------------------------------------------------------- slots
      if (elect_one()) {
        RsRing ring{0, 0};
        uint32_t used = 0;
        bool ok = true;
        for (int t = cluster; t < n_tiles && ok; t += n_clusters) {
          const MassTile tile = a.tiles[t];
          if (tile.count == 0 || seg0 >= tile.nv) continue;
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
          const MassTile tile = a.tiles[t];
          if (tile.count == 0 || seg0 >= tile.nv) continue;
          const int terms = stacked(tile) ? 1 : TERMS;
          for (int k0 = 0; k0 < nkb && ok; k0 += chunk, ++acc) {
            const uint32_t buf = acc & 1, use = acc >> 1;
            if (use > 0 && !(ok = mbar_wait_spin(&s.s_empty[buf], (use - 1) & 1))) break;
            tc_fence_after();
            const int k1 = min(nkb, k0 + chunk);
            for (int kb = k0; kb < k1; ++kb) {
              if (!(ok = mbar_wait_spin(&s.full[ring.st], ring.phase))) break;
              fence_proxy_async_smem();  // Q was written by this CTA's threads
              tc_fence_after();
              const uint32_t st = smem_u32(s.stages + ring.st * STAGE), bk = st + TERMS * MS_ATILE;
  #pragma unroll
              for (int ks = 0; ks < 4; ++ks)
  #pragma unroll
                for (int x = 0; x < TERMS; ++x)
                  if (x < terms) tc_mma<0>(taddr + buf * MS_N, umma_desc_k_sw128(st + x * MS_ATILE + ks * 32),
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
    } else if (warp >= 4) {
      // --------------------------------------------------------------------------------------------- rows of Q
      // Eight lanes a row (16 bytes each: chunk j of row r at chunk j ^ (r % 8)), 4 MS_PRODUCERS rows at a time.
      constexpr int STEP = 4 * MS_PRODUCERS, PASSES = MS_M / STEP;
      const int t0 = threadIdx.x - 128;
      const int sub = t0 >> 3, ch = t0 & 7;
      const char* q = static_cast<const char*>(a.q16);
      const int64_t row_bytes = (int64_t)a.d_s * 2, term_bytes = a.n_rows * row_bytes;
      RsRing ring{0, 0};
      uint32_t used = 0;
      bool ok = true;
      for (int t = cluster; t < n_tiles && ok; t += n_clusters) {
        const MassTile tile = a.tiles[t];
        if (tile.count == 0 || seg0 >= tile.nv) continue;
        const uint32_t term_at = stacked(tile) ? ms_few(TERMS) * 128 : MS_ATILE;
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
              if (TERMS >= 2) ms_copy16(dst + term_at, src + term_bytes, in ? 16 : 0);
              if (TERMS == 3) ms_copy16(dst + 2 * term_at, src + 2 * term_bytes, in ? 16 : 0);
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
    const int quarter = warp & 3, half = (warp - MS_LOW) >> 2;
    const int r = quarter * 32 + lane;               // pair of the tile = TMEM lane
    const uint32_t tl = taddr + ((uint32_t)(quarter * 32) << 16) + half * 128;
    const int n0 = seg0 + half * 128;                // first slot of this warp
    const int width = max(0, min(128, a.per - half * 128));
    uint32_t acc = 0, gen = 0;
    for (int t = cluster; t < n_tiles; t += n_clusters) {
      const MassTile tile = a.tiles[t];
      if (tile.count == 0) continue;
      const bool few = stacked(tile), here = r < tile.count, any = quarter * 32 < tile.count;
      const bool drain = (few ? (TERMS == 3 ? 0 : quarter & 1) : quarter) * 32 < tile.count && width > 0 &&
                         (TERMS < 3 || !few || quarter < 3);  // this warp's lanes hold sums
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
        for (int k0 = 0; k0 < nkb; k0 += chunk, ++acc) {
          const uint32_t buf = acc & 1;
          done(*s.abort_flag || mbar_wait_spin(&s.s_full[buf], (acc >> 1) & 1));
          tc_fence_after();
          if (drain) {
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
      if (TERMS == 2 && few && drain) {  // the lo rows' sums, 64 lanes further, to those of the hi rows
        float* x = s.xch + (half * MS_FEW + (quarter & 1) * 32 + lane) * MS_XPITCH;
#pragma unroll
        for (int g = 0; g < 128; g += 16) {
          if (quarter >= 2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = v[g + i];
          }
          named_bar_sync(2 + half * 2 + (quarter & 1), 64);
          if (quarter < 2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[g + i] += x[i];
          }
          named_bar_sync(2 + half * 2 + (quarter & 1), 64);
        }
      }
      if (TERMS == 3 && few && drain) {  // the mid and lo rows' sums, 32 and 64 lanes further
        float* x = s.xch + (half * MS_FEW + lane) * MS_XPITCH;
#pragma unroll
        for (int g = 0; g < 128; g += 16) {
          if (quarter > 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[(quarter - 1) * 32 * MS_XPITCH + i] = v[g + i];
          }
          named_bar_sync(2 + half, 96);
          if (quarter == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[g + i] += x[i] + x[32 * MS_XPITCH + i];
          }
          named_bar_sync(2 + half, 96);
        }
      }
      // e^(score - max) of this half, its maximum and sum
      float m = -CUDART_INF_F, l = 0.f;
      if (any) {
        float mx[4] = {m, m, m, m}, sum[4] = {0.f, 0.f, 0.f, 0.f};  // (four chains: the warps are few)
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i < nv) mx[i & 3] = fmaxf(mx[i & 3], v[i] * c);
        m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
#pragma unroll
        for (int i = 0; i < 128; ++i) {
          v[i] = i < nv ? pf_exp2(fmaf(v[i], c, -m)) : 0.f;
          sum[i & 3] += v[i];
        }
        l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      float* stat = s.stat + (size_t)(gen & 1) * cs * 2 * MS_M * 2;
      if (threadIdx.x == 32 * MS_LOW) mbar_arrive_expect_tx(&s.st[gen & 1], (uint32_t)cs * 2 * MS_M * 8);
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
        float sum = 0.f;
        if (any) {
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = g + i < nv ? v[g + i] * f : 0.f;  // (not 0 * NaN)
          sum = rs_reduce<32>(x, lane, [](float p, float q) { return p + q; });
        }
        s.cols[quarter * MS_N + half * 128 + g + lane] = sum;
      }
      named_bar_sync(1, 32 * MS_EPI);
      const int col = (int)threadIdx.x - 32 * MS_LOW;
      const bool mine = col < a.per && seg0 + col < a.page_rows;
      float sum = 0.f;
      if (mine) {
        sum = s.cols[col];
#pragma unroll
          for (int g = 1; g < 4; ++g) sum += s.cols[g * MS_N + col];
      }
      const int64_t at = (int64_t)tile.page * a.page_rows + seg0 + col;
      bool last = tile.total == 1;
      if (!last) {
        if (mine) a.part[(int64_t)t * a.page_rows + seg0 + col] = sum;
        __threadfence();
        named_bar_sync(1, 32 * MS_EPI);  // (the CTA's part of the tile is written; the column sums are read)
        if (col == 0) *s.last = atomicAdd(&a.done[tile.page * cs + rank], 1) == tile.total - 1;
        named_bar_sync(1, 32 * MS_EPI);
        last = *s.last;
        if (last && mine) {
          __threadfence();
          sum = 0.f;
          for (int j = 0; j < tile.total; ++j) {
            const int tj = j == tile.total - 1 && tile.few >= 0 ? tile.few : tile.base + j * tile.stride;
            sum += __ldcg(a.part + (int64_t)tj * a.page_rows + seg0 + col);
          }
        }
      }
      if (last && mine) a.mass[at] = a.prior ? fmaf(a.decay, a.prior[at], sum) : sum;
      named_bar_sync(1, 32 * MS_EPI);
      ++gen;
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

}  // namespace xencb
