// Eviction: the slots of every page that received most attention stay, in their order, at the front of the page; the others
// go. What goes by is mass [n_pages, page_rows] (read_mass), the same rows leave every pool (every depth, keys and values).
//
//   rows[p] = the most rows of page p that some table reads; rank = a row's place among them by (mass descending, row)
//   a budget per chunk    page p keeps the rows with rank < min(rows[p], new_rows, max(keep, floor)), keep the largest of
//                         the entries that name the page
//   a budget per Library  every page keeps its `floor` heaviest rows; what is left of a Library's budget (its own valid rows
//                         among those count) goes to its heaviest other rows with rank < new_rows, ties to the lower chunk,
//                         then to the lower row; a row stays if some Library keeps it
//
// evict_plan (one CTA over the tables), evict_rank (a CTA per page sorts its rows: 64-bit keys in shared memory), for
// Library budgets evict_budget (a CTA per Library: radix select of the last mass that stays, three passes of 11, 11 and
// 10 bits) and evict_list, then one launch moves the rows of all pools. Nothing is read back by the host.
#pragma once

#include "pages.cuh"

namespace xencb {

constexpr int EV_MAX_ROWS = 4096;  // rows of a page: their sort keys in shared memory, ranks in 16 bits
constexpr int EV_WORDS = EV_MAX_ROWS / 32;

struct EvictArgs {
  const int32_t* page_of;      // [n_lib, C]
  const int32_t* n_valid;      // [n_lib, C]
  const int32_t* n_chunks_of;  // [n_lib] or null
  int64_t n_lib;
  int C, n_pages, page_rows, new_rows;
  const float* mass;    // [n_pages, page_rows]
  const int32_t* keep;  // [n_lib, C], or [n_lib] with per_library, or null: keep_all
  int keep_all, per_library, floor;
  // outputs
  int32_t* n_valid_out;  // [n_lib, C]
  float* mass_out;       // [n_pages, new_rows]
  int32_t* kept;         // [n_pages, new_rows]: source rows ascending, -1 behind them
  // workspace
  int* rows;       // [n_pages]
  int* most;       // [n_pages]
  int* count;      // [n_pages]: rows that stay
  uint16_t* rank;  // [n_pages, page_rows] (per_library)
  uint32_t* bits;  // [n_pages, words] (per_library)
  int words;
};

// Larger masses have larger orders; -0 and 0 are one mass, NaN comes last.
__device__ __forceinline__ uint32_t ev_order(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int ev_chunks(const EvictArgs& a, int64_t lib) {
  return a.n_chunks_of ? max(0, min(a.n_chunks_of[lib], a.C)) : a.C;
}

__global__ void __launch_bounds__(PG_THREADS) evict_plan_kernel(const EvictArgs a) {
  pdl_trigger();
  for (int i = threadIdx.x; i < a.n_pages; i += PG_THREADS) {
    a.rows[i] = 0;
    a.most[i] = 0;
  }
  __syncthreads();
  const int64_t n = a.n_lib * a.C;
  for (int64_t e = threadIdx.x; e < n; e += PG_THREADS) {
    const int64_t lib = e / a.C;
    if ((int)(e - lib * a.C) >= ev_chunks(a, lib)) continue;
    const int p = a.page_of[e];
    if (p < 0 || p >= a.n_pages) {
      flag_error(XENCB_DEV_BADPAGE);
      continue;
    }
    const int nv = a.n_valid[e];
    if (nv > a.page_rows) flag_error(XENCB_DEV_CLAMPED);
    atomicMax(&a.rows[p], min(nv, a.page_rows));
    if (!a.per_library) atomicMax(&a.most[p], a.keep ? a.keep[e] : a.keep_all);
  }
}

// The list of a page's rows that stay and their masses, from the bits in shared memory. `sh` holds 32 ints.
__device__ __forceinline__ void ev_emit(const EvictArgs& a, int p, const uint32_t* bits, int* base) {
  // base: [words] exclusive counts, by the first warp
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int run = 0;
    for (int w0 = 0; w0 < a.words; w0 += 32) {
      const int c = w0 + lane < a.words ? __popc(bits[w0 + lane]) : 0;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (w0 + lane < a.words) base[w0 + lane] = run + incl - c;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) base[a.words] = run;
  }
  __syncthreads();
  const int total = min(base[a.words], a.new_rows);
  const float* m = a.mass + (int64_t)p * a.page_rows;
  int32_t* k = a.kept + (int64_t)p * a.new_rows;
  float* mo = a.mass_out + (int64_t)p * a.new_rows;
  for (int i = threadIdx.x; i < a.page_rows; i += blockDim.x) {
    const uint32_t w = bits[i >> 5];
    const int at = base[i >> 5] + __popc(w & ((1u << (i & 31)) - 1u));
    if (((w >> (i & 31)) & 1u) && at < total) {
      k[at] = i;
      mo[at] = m[i];
    }
  }
  for (int i = total + threadIdx.x; i < a.new_rows; i += blockDim.x) {
    k[i] = -1;
    mo[i] = 0.f;
  }
  if (threadIdx.x == 0) a.count[p] = total;
}

// One CTA per page, n2 / 2 threads (at least 64, at most 1024); dynamic shared memory: n2 keys, n2 a power of two.
__global__ void __launch_bounds__(1024) evict_rank_kernel(const EvictArgs a, int n2) {
  extern __shared__ unsigned long long ev_keys[];
  __shared__ uint32_t bits[EV_WORDS];
  __shared__ int base[EV_WORDS + 1];
  pdl_trigger();
  pdl_wait();
  const int p = blockIdx.x, n = a.rows[p];
  for (int i = threadIdx.x; i < a.words; i += blockDim.x) bits[i] = 0u;
  const int stay = min(min(n, a.new_rows), a.per_library ? a.floor : max(a.most[p], a.floor));
  if (n > 0) {
    const float* m = a.mass + (int64_t)p * a.page_rows;
    for (int i = threadIdx.x; i < n2; i += blockDim.x)
      ev_keys[i] = i < n ? ((unsigned long long)(~ev_order(m[i])) << 32) | (unsigned)i : ~0ull;
    for (int size = 2; size <= n2; size <<= 1)
      for (int step = size >> 1; step > 0; step >>= 1) {
        __syncthreads();
        for (int t = threadIdx.x; t < n2 / 2; t += blockDim.x) {
          const int i = 2 * t - (t & (step - 1)), j = i + step;
          const unsigned long long x = ev_keys[i], y = ev_keys[j];
          if ((x > y) == ((i & size) == 0)) {
            ev_keys[i] = y;
            ev_keys[j] = x;
          }
        }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int r = (int)(ev_keys[i] & 0xffffffffu);
      if (a.per_library) a.rank[(int64_t)p * a.page_rows + r] = (uint16_t)i;
      if (i < stay) atomicOr(&bits[r >> 5], 1u << (r & 31));
    }
  }
  __syncthreads();
  if (a.per_library) {
    for (int i = threadIdx.x; i < a.words; i += blockDim.x) a.bits[(int64_t)p * a.words + i] = bits[i];
    return;
  }
  ev_emit(a, p, bits, base);
}

// One CTA per Library.
__global__ void __launch_bounds__(PG_THREADS) evict_budget_kernel(const EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int sh[32];
  __shared__ int s_bin, s_left;
  pdl_trigger();
  pdl_wait();
  const int64_t lib = blockIdx.x;
  const int64_t n = (int64_t)ev_chunks(a, lib) * a.page_rows;
  // the row behind position i of the Library: its page, and whether it is read; -1 if not
  auto row = [&](int64_t i, int* r) -> int {
    const int64_t e = lib * a.C + i / a.page_rows;
    *r = (int)(i % a.page_rows);
    const int p = a.page_of[e];
    return p < 0 || p >= a.n_pages || *r >= a.n_valid[e] ? -1 : p;
  };
  auto at = [&](int p, int r) { return (int64_t)p * a.page_rows + r; };
  int first = 0, others = 0;
  for (int64_t i = threadIdx.x; i < n; i += PG_THREADS) {
    int r;
    const int p = row(i, &r);
    if (p < 0) continue;
    const int k = a.rank[at(p, r)];
    first += k < a.floor && k < a.new_rows;
    others += k >= a.floor && k < a.new_rows;
  }
  int n_first, n_others;
  pg_scan(first, sh, &n_first);
  pg_scan(others, sh, &n_others);
  int left = (a.keep ? a.keep[lib] : a.keep_all) - n_first;
  if (left <= 0 || n_others == 0) return;
  uint32_t last = 0;   // the order of the last mass that stays
  bool all = left >= n_others;
  if (!all) {
    const int shift[3] = {21, 10, 0}, width[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = threadIdx.x; i < 2048; i += PG_THREADS) hist[i] = 0;
      __syncthreads();
      const int s = shift[pass], nbins = 1 << width[pass];
      for (int64_t i = threadIdx.x; i < n; i += PG_THREADS) {
        int r;
        const int p = row(i, &r);
        if (p < 0) continue;
        const int k = a.rank[at(p, r)];
        if (k < a.floor || k >= a.new_rows) continue;
        const uint32_t o = ev_order(a.mass[at(p, r)]);
        if (pass > 0 && (o >> (s + width[pass])) != (last >> (s + width[pass]))) continue;
        atomicAdd(&hist[(o >> s) & (nbins - 1)], 1);
      }
      __syncthreads();
      // the bin, from the top, in which `left` runs out: thread t owns bins nbins - 1 - 2 t and the one below it
      const int b1 = nbins - 1 - 2 * (int)threadIdx.x, b0 = b1 - 1;
      const int c1 = b1 >= 0 ? hist[b1] : 0, c0 = b0 >= 0 ? hist[b0] : 0;
      int total;
      const int before = pg_scan(c1 + c0, sh, &total);
      if (before < left && left <= before + c1) { s_bin = b1; s_left = left - before; }
      else if (before + c1 < left && left <= before + c1 + c0) { s_bin = b0; s_left = left - before - c1; }
      __syncthreads();
      last |= (uint32_t)s_bin << s;
      left = s_left;
      __syncthreads();
    }
  }
  // heavier ones stay; `left` of those with the last mass, in the order of their chunks and rows
  int taken = 0;
  for (int64_t i0 = 0; i0 < n; i0 += PG_THREADS) {
    const int64_t i = i0 + threadIdx.x;
    int r = 0, p = -1;
    if (i < n) p = row(i, &r);
    uint32_t o = 0;
    bool may = false;
    if (p >= 0) {
      const int k = a.rank[at(p, r)];
      may = k >= a.floor && k < a.new_rows;
      o = ev_order(a.mass[at(p, r)]);
    }
    bool stays = may && (all || o > last);
    if (!all && taken < left) {
      int total;
      const bool tie = may && o == last;
      const int before = pg_scan(tie ? 1 : 0, sh, &total);
      stays = stays || (tie && taken + before < left);
      taken += total;
    }
    if (stays) atomicOr(&a.bits[(int64_t)p * a.words + (r >> 5)], 1u << (r & 31));
  }
}

__global__ void __launch_bounds__(256) evict_list_kernel(const EvictArgs a) {
  __shared__ uint32_t bits[EV_WORDS];
  __shared__ int base[EV_WORDS + 1];
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < a.words; i += blockDim.x) bits[i] = a.bits[(int64_t)blockIdx.x * a.words + i];
  __syncthreads();
  ev_emit(a, blockIdx.x, bits, base);
}

struct EvictPools {
  const char* src[PG_POOLS];
  char* dst[PG_POOLS];
  int64_t row_bytes[PG_POOLS];
  int first[PG_POOLS + 1];  // first slice of each pool's page in a page's list of slices
  int slices;
};

// The rows of each entry of the tables that stay: those of its page that lie before its own n_valid.
__device__ __forceinline__ void ev_tables(const EvictArgs& a) {
  const int64_t n = a.n_lib * a.C;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t lib = e / a.C;
    const int p = a.page_of[e];
    int left = 0;
    if ((int)(e - lib * a.C) < ev_chunks(a, lib) && p >= 0 && p < a.n_pages) {
      const int32_t* k = a.kept + (int64_t)p * a.new_rows;
      const int nv = a.n_valid[e];
      int hi = a.count[p];  // the first kept row at or past nv
      while (left < hi) {
        const int mid = (left + hi) >> 1;
        if (k[mid] < nv) left = mid + 1;
        else hi = mid;
      }
    }
    a.n_valid_out[e] = left;
  }
}

// Into new pools: a work item is a slice of one new page of one pool, EV_UNROLL units a thread, every load in flight
// before the first store. V: 16 bytes where every row is a multiple of it, else 2.
constexpr int EV_THREADS = 256;
constexpr int EV_UNROLL = 4;

template <typename V>
__global__ void __launch_bounds__(EV_THREADS) evict_gather_kernel(const EvictArgs a, const EvictPools pools) {
  pdl_wait();
  ev_tables(a);
  const int64_t n = (int64_t)a.n_pages * pools.slices;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const int p = (int)(w / pools.slices);
    int sl = (int)(w % pools.slices), k = 0;
    while (sl >= pools.first[k + 1]) ++k;
    sl -= pools.first[k];
    const unsigned upr = (unsigned)(pools.row_bytes[k] / sizeof(V));  // units of a row
    const int64_t units = (int64_t)upr * a.new_rows;
    const V* src = reinterpret_cast<const V*>(pools.src[k] + (int64_t)p * a.page_rows * pools.row_bytes[k]);
    V* dst = reinterpret_cast<V*>(pools.dst[k] + (int64_t)p * a.new_rows * pools.row_bytes[k]);
    const int32_t* kept = a.kept + (int64_t)p * a.new_rows;
    const int64_t at = (int64_t)sl * (EV_THREADS * EV_UNROLL) + threadIdx.x;
    V v[EV_UNROLL];
#pragma unroll
    for (int i = 0; i < EV_UNROLL; ++i) {
      const int64_t u = at + i * EV_THREADS;
      v[i] = pg_zero<V>();
      if (u < units) {
        const unsigned j = (unsigned)u / upr;  // (a page's units fit 31 bits)
        const int r = kept[j];
        if (r >= 0) v[i] = __ldcs(src + (int64_t)r * upr + ((unsigned)u - j * upr));
      }
    }
#pragma unroll
    for (int i = 0; i < EV_UNROLL; ++i)
      if (at + i * EV_THREADS < units) __stcs(dst + at + i * EV_THREADS, v[i]);
  }
}

// Within the pools: a thread owns one unit of every row of a page and walks the rows upwards, EV_ROWS loads in flight. A
// row moves to a lower place or stays, and no later load lies below a place that is already written. The rows between the
// last that stays and the last that was read become zeros; what lay behind them stays as it was.
constexpr int EV_ROWS = 8;

template <typename V>
__global__ void __launch_bounds__(EV_THREADS) evict_inplace_kernel(const EvictArgs a, const EvictPools pools) {
  pdl_wait();
  ev_tables(a);
  const int64_t n = (int64_t)a.n_pages * pools.slices;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const int p = (int)(w / pools.slices);
    int sl = (int)(w % pools.slices), k = 0;
    while (sl >= pools.first[k + 1]) ++k;
    sl -= pools.first[k];
    const unsigned upr = (unsigned)(pools.row_bytes[k] / sizeof(V));
    const unsigned u = (unsigned)sl * EV_THREADS + threadIdx.x;
    if (u >= upr) continue;
    V* page = reinterpret_cast<V*>(pools.dst[k] + (int64_t)p * a.page_rows * pools.row_bytes[k]) + u;
    const int32_t* kept = a.kept + (int64_t)p * a.new_rows;
    const int stay = a.count[p], rows = a.rows[p];
    for (int j0 = 0; j0 < stay; j0 += EV_ROWS) {
      V v[EV_ROWS];
      int r[EV_ROWS];
#pragma unroll
      for (int i = 0; i < EV_ROWS; ++i) {
        r[i] = j0 + i < stay ? kept[j0 + i] : -1;
        if (r[i] > j0 + i) v[i] = page[(int64_t)r[i] * upr];
      }
#pragma unroll
      for (int i = 0; i < EV_ROWS; ++i)
        if (r[i] > j0 + i) page[(int64_t)(j0 + i) * upr] = v[i];
    }
    for (int j = stay; j < rows; ++j) page[(int64_t)j * upr] = pg_zero<V>();
  }
}

}  // namespace xencb
