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
// evict_rank (a CTA per page ranks its rows), for Library budgets evict_budget (a CTA per Library: radix select of the last
// mass that stays, three passes of 11, 11 and 10 bits over keys in shared memory), then one launch moves the rows of all
// pools. What stays is handed on as one bit a row. A page's CTA looks through the tables itself where they are short;
// evict_plan does it for long ones. Nothing is read back by the host.
//
// HBM bounds the move: 121 pages of 128 of 512 rows in four pools of 4 KiB rows into pages of 128 (0.52 GB) takes 80 us,
// 6.5 TB/s. The ranks take 10 us there (a row's comparisons with 511 others), 5 on pages of 64; the budgets of 5 Libraries
// of 37 chunks of 203 rows 13 (latency: a CTA each, three passes over the keys). Within the pools the same eviction takes
// 230 us: it writes zeros into the 0.76 GB that the rows which went leave, 5.5 TB/s with the rows that move.
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
  int direct;  // the pages' CTAs look through the tables
  // workspace
  int* rows;       // [n_pages]
  int* most;       // [n_pages] (with a plan)
  uint32_t* bits;  // [n_pages, words]: the rows that stay
  uint32_t* keys;  // [n_pages, page_rows] (per_library): EV_FIRST, a mass's order, or 0: not to be had
  int words;
};
constexpr uint32_t EV_FIRST = 0xffffffffu;  // one of the page's `floor` heaviest rows

// Larger masses have larger orders (none is 0 or EV_FIRST); -0 and 0 are one mass, NaN comes last.
__device__ __forceinline__ uint32_t ev_order(float x) {
  if (x != x) return 1u;
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

// One CTA per page; dynamic shared memory: n2 orders, or 64-bit keys for pages of more than EV_COUNTED rows (n2 a power
// of two, at least page_rows). Up to EV_COUNTED rows a row's rank is counted, one thread a row; longer pages are sorted.
constexpr int EV_COUNTED = 512;
__global__ void __launch_bounds__(1024) evict_rank_kernel(const EvictArgs a, int n2) {
  extern __shared__ __align__(16) unsigned long long ev_keys[];
  __shared__ uint32_t bits[EV_WORDS];
  __shared__ int sh_rows, sh_most;
  pdl_trigger();
  const int p = blockIdx.x;
  if (threadIdx.x == 0) sh_rows = sh_most = 0;
  for (int i = threadIdx.x; i < a.words; i += blockDim.x) bits[i] = 0u;
  if (a.direct) {
    __syncthreads();
    const int64_t n = a.n_lib * a.C;
    for (int64_t e = threadIdx.x; e < n; e += blockDim.x) {
      const int64_t lib = e / a.C;
      if ((int)(e - lib * a.C) >= ev_chunks(a, lib)) continue;
      const int page = a.page_of[e], nv = a.n_valid[e];
      if (p == 0 && (page < 0 || page >= a.n_pages)) flag_error(XENCB_DEV_BADPAGE);
      if (page != p) continue;
      if (nv > a.page_rows) flag_error(XENCB_DEV_CLAMPED);
      atomicMax(&sh_rows, min(nv, a.page_rows));
      if (!a.per_library) atomicMax(&sh_most, a.keep ? a.keep[e] : a.keep_all);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.rows[p] = sh_rows;
  } else {
    pdl_wait();
    if (threadIdx.x == 0) {
      sh_rows = a.rows[p];
      sh_most = a.most[p];
    }
    __syncthreads();
  }
  const int n = sh_rows;
  const int stay = min(min(n, a.new_rows), a.per_library ? a.floor : max(sh_most, a.floor));
  const float* m = a.mass + (int64_t)p * a.page_rows;
  auto place = [&](int row, int rank, uint32_t order) {
    if (rank < stay) atomicOr(&bits[row >> 5], 1u << (row & 31));
    if (a.per_library)
      a.keys[(int64_t)p * a.page_rows + row] = rank < stay ? EV_FIRST : rank < a.new_rows ? order : 0u;
  };
  if (n2 <= EV_COUNTED) {
    uint32_t* o = reinterpret_cast<uint32_t*>(ev_keys);
    const int i = threadIdx.x;  // (n2 threads)
    const uint32_t mine = i < n ? ev_order(m[i]) : 0u;
    o[i] = mine;
    __syncthreads();
    if ((i & ~31) < n) {
      const uint4* o4 = reinterpret_cast<const uint4*>(o);
      const int w0 = (i & ~31) / 4, w1 = w0 + 8, end = (n + 3) / 4;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < w0; ++j) {  // equal ones before this row count
        const uint4 x = o4[j];
        rank += (x.x >= mine) + (x.y >= mine) + (x.z >= mine) + (x.w >= mine);
      }
#pragma unroll
      for (int j = w0 * 4; j < w1 * 4; ++j) rank += o[j] > mine || (o[j] == mine && j < i);
#pragma unroll 4
      for (int j = w1; j < end; ++j) {
        const uint4 x = o4[j];
        rank += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
      }
      if (i < n) place(i, rank, mine);
    }
  } else if (n > 0) {
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
    for (int i = threadIdx.x; i < n; i += blockDim.x)
      place((int)(ev_keys[i] & 0xffffffffu), i, ~(uint32_t)(ev_keys[i] >> 32));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.words; i += blockDim.x) a.bits[(int64_t)p * a.words + i] = bits[i];
}

// One CTA per Library. Its keys, chunk by chunk in rows of `pitch`, lie in shared memory (cached), or are read again in
// every pass.
template <bool CACHED>
__global__ void __launch_bounds__(PG_THREADS) evict_budget_kernel(const EvictArgs a, int pitch) {
  extern __shared__ uint32_t ev_cache[];
  __shared__ int hist[2048];
  __shared__ int sh[32];
  __shared__ int s_bin, s_left, s_ties;
  pdl_trigger();
  pdl_wait();
  const int64_t lib = blockIdx.x;
  const int C = ev_chunks(a, lib);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rounds = (a.page_rows + 31) / 32;
  // warp w takes chunks w, w + 32, ..., 32 rows at a time: f(chunk, page, round, key); rows that are not read have key 0
  auto each = [&](auto f, bool cached) {
    for (int c = warp; c < C; c += 32) {
      const int64_t e = lib * a.C + c;
      const int p = a.page_of[e], nv = min(a.n_valid[e], a.page_rows);
      const bool ok = p >= 0 && p < a.n_pages;
#pragma unroll 4
      for (int w = 0; w < rounds; ++w) {
        const int r = w * 32 + lane;
        uint32_t key = 0u;
        if (cached) key = ev_cache[c * pitch + r];
        else if (ok && r < nv) key = a.keys[(int64_t)p * a.page_rows + r];
        f(c, p, w, key);
      }
    }
  };
  int first = 0, others = 0;
  each([&](int c, int, int w, uint32_t key) {
    if (CACHED) ev_cache[c * pitch + w * 32 + lane] = key;
    first += key == EV_FIRST;
    others += key != EV_FIRST && key != 0u;
  }, false);
  __syncwarp();
  int n_first, n_others;
  pg_scan(first, sh, &n_first);
  pg_scan(others, sh, &n_others);
  int left = max(0, a.keep ? a.keep[lib] : a.keep_all) - n_first;
  if (left <= 0 || n_others == 0) return;
  uint32_t last = 1u;  // the order of the last mass that stays
  bool cut = false;    // not all of that mass stay
  if (left < n_others) {
    last = 0u;
    const int shift[3] = {21, 10, 0}, width[3] = {11, 11, 10};
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = threadIdx.x; i < 2048; i += PG_THREADS) hist[i] = 0;
      __syncthreads();
      const int s = shift[pass], nbins = 1 << width[pass];
      each([&](int, int, int, uint32_t key) {
        const bool in = key != 0u && key != EV_FIRST &&
                        (pass == 0 || (key >> (s + width[pass])) == (last >> (s + width[pass])));
        if (in) atomicAdd(&hist[(key >> s) & (nbins - 1)], 1);
      }, CACHED);
      __syncthreads();
      // the bin, from the top, in which `left` runs out: thread t owns bins nbins - 1 - 2 t and the one below it
      const int b1 = nbins - 1 - 2 * (int)threadIdx.x, b0 = b1 - 1;
      const int c1 = b1 >= 0 ? hist[b1] : 0, c0 = b0 >= 0 ? hist[b0] : 0;
      int total;
      const int before = pg_scan(c1 + c0, sh, &total);
      if (before < left && left <= before + c1) { s_bin = b1; s_left = left - before; s_ties = c1; }
      else if (before + c1 < left && left <= before + c1 + c0) { s_bin = b0; s_left = left - before - c1; s_ties = c0; }
      __syncthreads();
      last |= (uint32_t)s_bin << s;
      left = s_left;
      cut = s_ties > left;
      __syncthreads();
    }
  }
  each([&](int, int p, int w, uint32_t key) {
    const uint32_t stays = __ballot_sync(0xffffffffu, key != EV_FIRST && key != 0u && (cut ? key > last : key >= last));
    if (lane == 0 && stays) atomicOr(&a.bits[(int64_t)p * a.words + w], stays);
  }, CACHED);
  if (!cut) return;
  // `left` of those with the last mass, in the order of their chunks and rows
  const int64_t n = (int64_t)C * a.page_rows;
  for (int64_t i0 = 0, taken = 0; i0 < n && taken < left; i0 += PG_THREADS) {
    const int64_t i = i0 + threadIdx.x;
    int p = -1, r = 0;
    bool tie = false;
    if (i < n) {
      const int64_t e = lib * a.C + i / a.page_rows;
      r = (int)(i % a.page_rows);
      p = a.page_of[e];
      tie = p >= 0 && p < a.n_pages && r < a.n_valid[e] && a.keys[(int64_t)p * a.page_rows + r] == last;
    }
    int total;
    const int before = pg_scan(tie ? 1 : 0, sh, &total);
    if (tie && taken + before < left) atomicOr(&a.bits[(int64_t)p * a.words + (r >> 5)], 1u << (r & 31));
    taken += total;
  }
}

struct EvictPools {
  const char* src[PG_POOLS];
  char* dst[PG_POOLS];
  int64_t row_bytes[PG_POOLS];
  int first[PG_POOLS + 1];  // first slice of each pool's page in a page's list of slices
  int slices;
  int outputs;  // this launch writes n_valid_out, mass_out and kept too
};

// The rows of each entry of the tables that stay: those of its page that lie before its own n_valid.
__device__ __forceinline__ void ev_tables(const EvictArgs& a) {
  const int64_t n = a.n_lib * a.C;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t lib = e / a.C;
    const int p = a.page_of[e], nv = min(a.n_valid[e], a.page_rows);
    int left = 0;
    if ((int)(e - lib * a.C) < ev_chunks(a, lib) && p >= 0 && p < a.n_pages)
      for (int w = 0; w * 32 < nv; ++w) {
        const uint32_t u = a.bits[(int64_t)p * a.words + w];
        left += __popc(nv - w * 32 >= 32 ? u : u & ((1u << (nv - w * 32)) - 1u));
      }
    a.n_valid_out[e] = left;
  }
}

// The rows of page p that stay, ascending, into list; returns their number. By all threads of the CTA.
__device__ __forceinline__ int ev_list(const EvictArgs& a, int p, uint16_t* list, uint32_t* bits, int* base) {
  __syncthreads();  // (the list before is done with)
  for (int i = threadIdx.x; i < a.words; i += blockDim.x) bits[i] = a.bits[(int64_t)p * a.words + i];
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
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
  for (int i = threadIdx.x; i < a.page_rows; i += blockDim.x) {
    const uint32_t w = bits[i >> 5];
    const int at = base[i >> 5] + __popc(w & ((1u << (i & 31)) - 1u));
    if ((w >> (i & 31)) & 1u) list[at] = (uint16_t)i;
  }
  __syncthreads();
  return base[a.words];
}

// A page's share of mass_out and kept.
__device__ __forceinline__ void ev_outputs(const EvictArgs& a, int p, const uint16_t* list, int stay) {
  for (int j = threadIdx.x; j < a.new_rows; j += blockDim.x) {
    const int r = j < stay ? list[j] : -1;
    a.kept[(int64_t)p * a.new_rows + j] = r;
    a.mass_out[(int64_t)p * a.new_rows + j] = r >= 0 ? a.mass[(int64_t)p * a.page_rows + r] : 0.f;
  }
}

// Into new pools: a work item is a slice of one new page of one pool, EV_UNROLL units a thread, every load in flight
// before the first store. V: 16 bytes where every row is a multiple of it, else 2. A CTA takes consecutive items, so that
// it seldom needs another page's list.
constexpr int EV_THREADS = 256;
constexpr int EV_UNROLL = 4;

template <typename V>
__global__ void __launch_bounds__(EV_THREADS) evict_gather_kernel(const EvictArgs a, const EvictPools pools) {
  __shared__ uint16_t list[EV_MAX_ROWS];
  __shared__ uint32_t bits[EV_WORDS];
  __shared__ int base[EV_WORDS + 1];
  pdl_wait();
  if (pools.outputs) ev_tables(a);
  const int64_t n = (int64_t)a.n_pages * pools.slices;
  const int64_t per = (n + gridDim.x - 1) / gridDim.x, end = min(n, (int64_t)(blockIdx.x + 1) * per);
  int at_page = -1, stay = 0;
  for (int64_t w = blockIdx.x * per; w < end; ++w) {
    const int p = (int)(w / pools.slices);
    int sl = (int)(w % pools.slices), k = 0;
    if (p != at_page) {
      stay = ev_list(a, p, list, bits, base);
      at_page = p;
    }
    if (sl == 0 && pools.outputs) ev_outputs(a, p, list, stay);
    while (sl >= pools.first[k + 1]) ++k;
    sl -= pools.first[k];
    const unsigned upr = (unsigned)(pools.row_bytes[k] / sizeof(V));  // units of a row
    const unsigned units = upr * (unsigned)a.new_rows;                // (a page's units fit 31 bits)
    const V* src = reinterpret_cast<const V*>(pools.src[k] + (int64_t)p * a.page_rows * pools.row_bytes[k]);
    V* dst = reinterpret_cast<V*>(pools.dst[k] + (int64_t)p * a.new_rows * pools.row_bytes[k]);
    const unsigned at = (unsigned)sl * (EV_THREADS * EV_UNROLL) + threadIdx.x;
    V v[EV_UNROLL];
#pragma unroll
    for (int i = 0; i < EV_UNROLL; ++i) {
      const unsigned u = at + i * EV_THREADS;
      v[i] = pg_zero<V>();
      if (u < units) {
        const unsigned j = u / upr;
        if ((int)j < stay) v[i] = __ldcs(src + (int64_t)list[j] * upr + (u - j * upr));
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
  __shared__ uint16_t list[EV_MAX_ROWS];
  __shared__ uint32_t bits[EV_WORDS];
  __shared__ int base[EV_WORDS + 1];
  pdl_wait();
  if (pools.outputs) ev_tables(a);
  const int64_t n = (int64_t)a.n_pages * pools.slices;
  for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const int p = (int)(w / pools.slices);
    int sl = (int)(w % pools.slices), k = 0;
    const int stay = ev_list(a, p, list, bits, base), rows = a.rows[p];
    if (sl == 0 && pools.outputs) ev_outputs(a, p, list, stay);
    while (sl >= pools.first[k + 1]) ++k;
    sl -= pools.first[k];
    const unsigned upr = (unsigned)(pools.row_bytes[k] / sizeof(V));
    const unsigned u = (unsigned)sl * EV_THREADS + threadIdx.x;
    if (u >= upr) continue;
    V* page = reinterpret_cast<V*>(pools.dst[k] + (int64_t)p * a.page_rows * pools.row_bytes[k]) + u;
    for (int j0 = 0; j0 < stay; j0 += EV_ROWS) {
      V v[EV_ROWS];
      int r[EV_ROWS];
#pragma unroll
      for (int i = 0; i < EV_ROWS; ++i) {
        r[i] = j0 + i < stay ? list[j0 + i] : -1;
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
