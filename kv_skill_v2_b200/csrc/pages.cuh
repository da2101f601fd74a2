// Page operators of a slot pool that several Libraries share: forking (a child's table names its parent's pages up
// to a chunk, and fresh copies behind it) and compacting (live pages moved to the front). A page is live when some
// table names it; a Library is freed by dropping its table.
//
// One plan kernel (a single CTA: the tables are a few thousand integers) marks the live pages in a bitmap in shared
// memory, ranks them with a block scan and writes the new tables and the list of page copies; one copy kernel then
// moves the rows of every pool (every depth, keys and values) in one launch. Nothing is read back by the host: the
// number of copies stays on the device.
#pragma once

#include "common.cuh"

namespace xencb {

constexpr int PG_THREADS = 1024;
constexpr int PG_POOLS = 32;  // pools per copy launch
constexpr int PG_MAX_PAGES = 1 << 20;  // the live bitmap (128 KiB) fits shared memory

struct PageMove {
  int src, dst, rows;  // rows < 0: nothing to copy
};

struct PagePlanArgs {
  const int32_t* page_of;      // [n_lib, C]
  const int32_t* n_valid;      // [n_lib, C]
  const int32_t* n_chunks_of;  // [n_lib] or null
  int64_t n_lib;
  int C;
  int n_pages, page_rows;
  // fork
  const int32_t* parents;   // [m]
  const int32_t* own_from;  // [m]
  int64_t m;
  // outputs
  int32_t* table;  // fork: [m, C]; compact: [n_lib, C]
  int32_t* count;  // fork: fresh pages that were missing; compact: live pages
  // workspace
  PageMove* moves;
  int* n_moves;
  int* list;  // fork: free pages in ascending order; compact: holes below n_live
  int* to;    // compact: new place of a page
  int* rows;  // compact: valid rows of a page
};

// Exclusive block scan of one int per thread; *total gets the sum. `sh` holds PG_THREADS / 32 ints.
__device__ __forceinline__ int pg_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();
  if (lane == 31) sh[wid] = incl;
  __syncthreads();
  int w = sh[lane], wi = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) wi += y;
  }
  *total = __shfl_sync(0xffffffffu, wi, 31);
  return incl - v + __shfl_sync(0xffffffffu, wi - w, wid);
}

__device__ __forceinline__ int pg_chunks(const PagePlanArgs& a, int64_t lib) {
  return a.n_chunks_of ? max(0, min(a.n_chunks_of[lib], a.C)) : a.C;
}

__device__ __forceinline__ int pg_rows(const PagePlanArgs& a, int64_t e) {
  const int nv = a.n_valid[e];
  if (nv > a.page_rows) flag_error(XENCB_DEV_CLAMPED);
  return max(0, min(nv, a.page_rows));
}

// The live pages as bits; entries outside the pool are flagged and name nothing.
__device__ __forceinline__ void pg_mark_live(const PagePlanArgs& a, uint32_t* bits, int n_words, bool want_rows) {
  for (int i = threadIdx.x; i < n_words; i += PG_THREADS) bits[i] = 0u;
  if (want_rows)
    for (int i = threadIdx.x; i < a.n_pages; i += PG_THREADS) a.rows[i] = 0;
  __syncthreads();
  const int64_t n = a.n_lib * a.C;
  for (int64_t e = threadIdx.x; e < n; e += PG_THREADS) {
    const int64_t lib = e / a.C;
    if ((int)(e - lib * a.C) >= pg_chunks(a, lib)) continue;
    const int p = a.page_of[e];
    if (p < 0 || p >= a.n_pages) {
      flag_error(XENCB_DEV_BADPAGE);
      continue;
    }
    atomicOr(&bits[p >> 5], 1u << (p & 31));
    if (want_rows) atomicMax(&a.rows[p], pg_rows(a, e));
  }
  __syncthreads();
}

// bits of word i that are pages of the pool
__device__ __forceinline__ uint32_t pg_word_mask(int i, int n_pages) {
  const int left = n_pages - i * 32;
  return left >= 32 ? 0xffffffffu : (1u << left) - 1u;
}

__global__ void __launch_bounds__(PG_THREADS) pages_fork_plan_kernel(const PagePlanArgs a) {
  extern __shared__ uint32_t pg_bits[];
  __shared__ int sh[32];
  pdl_trigger();  // (the copy kernel waits for this grid before it reads the list)
  const int n_words = (a.n_pages + 31) / 32;
  pg_mark_live(a, pg_bits, n_words, false);
  // entries that need a fresh page, in (child, chunk) order: each thread owns a contiguous range
  const int64_t n = a.m * a.C;
  const int64_t per = (n + PG_THREADS - 1) / PG_THREADS;
  const int64_t e0 = min(n, (int64_t)threadIdx.x * per), e1 = min(n, e0 + per);
  // the parent's page when entry e of the children is a chunk of a known parent, else -1 (beyond the parent's chunks)
  // or -2 (bad parent or page)
  auto source = [&](int64_t e, int64_t* pe) -> int {
    const int64_t i = e / a.C;
    const int c = (int)(e - i * a.C);
    const int64_t parent = a.parents[i];
    if (parent < 0 || parent >= a.n_lib) return -2;
    if (c >= pg_chunks(a, parent)) return -1;
    *pe = parent * a.C + c;
    const int p = a.page_of[*pe];
    return p < 0 || p >= a.n_pages ? -2 : p;
  };
  int need = 0;
  for (int64_t e = e0; e < e1; ++e) {
    int64_t pe = 0;
    need += source(e, &pe) >= 0 && (int)(e % a.C) >= a.own_from[e / a.C];
  }
  int total = 0;
  const int first = pg_scan(need, sh, &total);
  // the first `total` free pages, ascending
  const int wper = (n_words + PG_THREADS - 1) / PG_THREADS;
  const int w0 = min(n_words, (int)threadIdx.x * wper), w1 = min(n_words, w0 + wper);
  int n_free = 0;
  for (int i = w0; i < w1; ++i) n_free += __popc(~pg_bits[i] & pg_word_mask(i, a.n_pages));
  int all_free = 0;
  int rank = pg_scan(n_free, sh, &all_free);
  for (int i = w0; i < w1 && rank < total; ++i)
    for (uint32_t f = ~pg_bits[i] & pg_word_mask(i, a.n_pages); f && rank < total; f &= f - 1, ++rank)
      a.list[rank] = i * 32 + __ffs(f) - 1;
  if (threadIdx.x == 0) {
    *a.count = max(0, total - all_free);
    *a.n_moves = min(total, all_free);
  }
  __syncthreads();  // (also orders the list's global writes within this CTA)
  int at = first;
  for (int64_t e = e0; e < e1; ++e) {
    int64_t pe = 0;
    int p = source(e, &pe);
    if (p == -2) {
      flag_error(XENCB_DEV_BADPAGE);
      p = -1;
    } else if (p == -1) {
      p = 0;  // chunk slots past a Library's own count name page 0, as PagedLibrary lays them out
    } else if ((int)(e % a.C) >= a.own_from[e / a.C]) {
      const int dst = at < all_free ? a.list[at] : -1;
      if (dst >= 0) a.moves[at] = PageMove{p, dst, pg_rows(a, pe)};
      ++at;
      p = dst;
    }
    a.table[e] = p;
  }
}

__global__ void __launch_bounds__(PG_THREADS) pages_compact_plan_kernel(const PagePlanArgs a) {
  extern __shared__ uint32_t pg_bits[];
  __shared__ int sh[32];
  pdl_trigger();  // (the copy kernel waits for this grid before it reads the list)
  const int n_words = (a.n_pages + 31) / 32;
  pg_mark_live(a, pg_bits, n_words, true);
  const int wper = (n_words + PG_THREADS - 1) / PG_THREADS;
  const int w0 = min(n_words, (int)threadIdx.x * wper), w1 = min(n_words, w0 + wper);
  int mine = 0;
  for (int i = w0; i < w1; ++i) mine += __popc(pg_bits[i]);
  int n_live = 0;
  const int first = pg_scan(mine, sh, &n_live);
  // live pages below n_live stay; the j-th live page at or above it goes to the j-th hole below it
  int stay = 0;
  for (int i = w0; i < w1; ++i)
    for (uint32_t b = pg_bits[i]; b; b &= b - 1) stay += i * 32 + __ffs(b) - 1 < n_live;
  int n_stay = 0;
  pg_scan(stay, sh, &n_stay);
  int rank = first;
  for (int i = w0; i < w1; ++i) {
    const uint32_t live = pg_bits[i];
    for (uint32_t f = ~live & pg_word_mask(i, a.n_pages); f; f &= f - 1) {
      const int p = i * 32 + __ffs(f) - 1;
      if (p < n_live) a.list[p - (rank + __popc(live & ((1u << (p & 31)) - 1u)))] = p;
    }
    rank += __popc(live);
  }
  __syncthreads();
  rank = first;
  for (int i = w0; i < w1; ++i)
    for (uint32_t b = pg_bits[i]; b; b &= b - 1, ++rank) {
      const int p = i * 32 + __ffs(b) - 1;
      if (p < n_live) {
        a.to[p] = p;
      } else {
        const int j = rank - n_stay;
        a.to[p] = a.list[j];
        a.moves[j] = PageMove{p, a.list[j], a.rows[p]};
      }
    }
  if (threadIdx.x == 0) {
    *a.count = n_live;
    *a.n_moves = n_live - n_stay;
  }
  __syncthreads();
  const int64_t n = a.n_lib * a.C;
  for (int64_t e = threadIdx.x; e < n; e += PG_THREADS) {
    const int64_t lib = e / a.C;
    const int p = a.page_of[e];
    int t = p;  // an entry outside the pool stays what it was
    if ((int)(e - lib * a.C) >= pg_chunks(a, lib)) t = 0;
    else if (p >= 0 && p < a.n_pages) t = a.to[p];
    a.table[e] = t;
  }
}

struct PagePools {
  char* base[PG_POOLS];
  int64_t row_bytes[PG_POOLS];
  int first[PG_POOLS + 1];  // first slice of each pool's page in a move's list of slices
  int slices;
  int page_rows;
};

// Copies the listed pages in every pool: the first `rows` rows of page src, then zeros to the end of the page. V is
// the unit of the accesses: 16 bytes where every pool's pages are 16-byte aligned, else 2 bytes (every slot type has
// at least two). A work item is a slice of one page of one pool, PG_UNROLL units a thread with every load in flight
// before the first store; the pages are read and written once, so both bypass L1. HBM bounds it: 64 pages of 2 MiB in
// four pools (0.94 GB read and written) 171 to 181 us with the plan, 5.2 to 5.5 TB/s, 0.79 to 0.84 of a plain copy's rate. 16 KiB slices on
// up to 64 CTAs per SM, most of which take a few slices: 8 units a thread on 8 CTAs per SM took 206 us.
constexpr int PG_COPY_THREADS = 256;
constexpr int PG_UNROLL = 4;

template <typename V> __device__ __forceinline__ V pg_zero();
template <> __device__ __forceinline__ uint4 pg_zero<uint4>() { return make_uint4(0u, 0u, 0u, 0u); }
template <> __device__ __forceinline__ uint16_t pg_zero<uint16_t>() { return 0; }

template <typename V>
__global__ void __launch_bounds__(PG_COPY_THREADS) pages_copy_kernel(const PagePools pools,
                                                                     const PageMove* __restrict__ moves,
                                                                     const int* __restrict__ n_moves) {
  constexpr int SLICE = PG_COPY_THREADS * PG_UNROLL * (int)sizeof(V);
  pdl_wait();
  const int64_t n = (int64_t)*n_moves * pools.slices;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const PageMove mv = moves[w / pools.slices];
    int sl = (int)(w % pools.slices), k = 0;
    while (sl >= pools.first[k + 1]) ++k;
    sl -= pools.first[k];
    const int64_t page_bytes = pools.row_bytes[k] * pools.page_rows;
    const int64_t keep = pools.row_bytes[k] * mv.rows;
    const char* src = pools.base[k] + mv.src * page_bytes;
    char* dst = pools.base[k] + mv.dst * page_bytes;
    const int64_t at = (int64_t)sl * SLICE + threadIdx.x * sizeof(V);
    V v[PG_UNROLL];
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      const int64_t o = at + (int64_t)i * PG_COPY_THREADS * sizeof(V);
      v[i] = o < keep ? __ldcs(reinterpret_cast<const V*>(src + o)) : pg_zero<V>();
    }
#pragma unroll
    for (int i = 0; i < PG_UNROLL; ++i) {
      const int64_t o = at + (int64_t)i * PG_COPY_THREADS * sizeof(V);
      if (o < keep && o + (int64_t)sizeof(V) > keep)  // the unit that holds the last valid bytes
        for (int b = (int)(keep - o); b < (int)sizeof(V); ++b) reinterpret_cast<char*>(&v[i])[b] = 0;
      if (o < page_bytes) __stcs(reinterpret_cast<V*>(dst + o), v[i]);
    }
  }
}

}  // namespace xencb
