// Low-rank adapters beside the interface projections: y = x W^T + s_a (x A_a^T) B_a^T, where a = adapter_of[row /
// rows_per_adapter] (negative: none) picks one of n adapters A [n, r, d_in], B [n, d_out, r], s [n].
//
// The projection's row kernels sum split partials of the GEMM, so the low-rank term is one more partial: shrink
// t = x A_a^T, then expand s_a t B_a^T into the slice behind the GEMM's. It lies before 1/rms, the bias, the norms
// and the gate, as the GEMM's partials do, and is float32 throughout.
//
// Two forms of each. Rows: one CTA per row (decode: every row has its own adapter, and the adapters' bytes bound it).
// Tiles: 64 rows of one adapter at a time, A and B read once a tile (prompts; the multiplications bound it), from
// AD_MIN_TILE rows per adapter on. Both forms, us a call of project_in (4096 -> 2048, 512 rows; rows / tiles):
//   rows per adapter             4          8          16         64
//   bf16 rows, rank 16         86 / 133   86 / 100   86 / 84    86 / 88
//   bf16 rows, rank 64        258 / 205  254 / 145  252 / 111  250 / 109
//   float32 rows, rank 16      88 / 211   88 / 153   88 / 115   88 / 143
//   float32 rows, rank 64     260 / 358  256 / 238  254 / 168  256 / 166
//
// Measured beside the projection (d_in 4096 -> 2048): 64 rows with 64 adapters of rank 16, shrink 10.6 us and expand
// 5.3 us of a call of 32.5 us (the GEMM 12.4 us); 2048 rows of 4 adapters of rank 32 (5120 -> 2048), shrink 19 us
// (78 us with float32 multiplications) and expand 27 us of 266 us; by rows the same took 159 and 249 us.
#pragma once

#include "gemm_f16x3.cuh"

namespace xencb {

constexpr int AD_MAX_RANK = 256;
constexpr int AD_TILE_ROWS = 64;   // rows of one adapter per tile
constexpr int AD_MIN_TILE = 16;    // rows per adapter from which tiles are used
constexpr int AD_TILE_J = 32;      // shrink: ranks per CTA
constexpr int AD_TILE_N = 128;     // expand: output columns per CTA
constexpr int AD_BK = 32;
constexpr int AD_MAX_SPLITS = 8;   // shrink: splits of d_in
constexpr int AD_KPS = 1280;       // columns of d_in per split of the projection GEMM at most

struct AdaptArgs {
  const void* a;        // [n, r, d_in]
  const void* b;        // [n, d_out, r]
  const float* scale;   // [n] or null (1)
  const int32_t* of;    // [ceil(n_rows / rows_per_adapter)]
  int64_t rows_per_adapter;
  int n, r, d_in, d_out;
  float* t;             // [splits, n_rows, r]
  int64_t n_rows;
  int splits;
  int vec_in, vec_r;    // rows of x and A (of B) are 16-byte aligned
};

// the adapter of a row, or -1; an index past the last adapter is flagged and read as none
__device__ __forceinline__ int ad_of(const AdaptArgs& p, int64_t row) {
  const int a = p.of[row / p.rows_per_adapter];
  if (a >= p.n) flag_error(XENCB_DEV_BADADAPTER);
  return a < 0 || a >= p.n ? -1 : a;
}

// ------------------------------------------------------------------------------------------------ rows
// t[row][j] = x[row] . A[a][j]: one warp per (row, j), 16-byte loads, four in flight.
template <typename TX, typename TA>
__global__ void __launch_bounds__(256) adapt_shrink_row_kernel(const TX* __restrict__ x, const AdaptArgs p) {
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int ad = ad_of(p, row);
  const int lane = threadIdx.x & 31, j = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (ad < 0 || j >= p.r) return;
  const TA* a = static_cast<const TA*>(p.a) + ((int64_t)ad * p.r + j) * p.d_in;
  const TX* xr = x + row * p.d_in;
  float s = 0.f;
  if (p.vec_in) {
    float s8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = lane * 8; k < p.d_in; k += 256) {
      float u[8], v[8];
      load8_f32<TX>(xr + k, u);
      load8_f32<TA>(a + k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s8[e] = fmaf(u[e], v[e], s8[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s += s8[e];
  } else {
    for (int k = lane; k < p.d_in; k += 32) s = fmaf(to_f32(xr[k]), to_f32(a[k]), s);
  }
  s = warp_sum(s);
  if (lane == 0) p.t[row * p.r + j] = s;
}

// out[row][n] = s_a sum_j t[row][j] B[a][n][j]; 0 for a row without an adapter. One thread per output.
template <typename TA>
__global__ void __launch_bounds__(256) adapt_expand_row_kernel(const AdaptArgs p, float* __restrict__ out) {
  __shared__ float t[AD_MAX_RANK];
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int ad = ad_of(p, row);
  if (ad >= 0)
    for (int j = threadIdx.x; j < p.r; j += 256) t[j] = p.t[row * p.r + j];
  __syncthreads();
  const int n = blockIdx.y * 256 + threadIdx.x;
  if (n >= p.d_out) return;
  float s = 0.f;
  if (ad >= 0) {
    const TA* b = static_cast<const TA*>(p.b) + ((int64_t)ad * p.d_out + n) * p.r;
    if (p.vec_r) {
#pragma unroll 2
      for (int j = 0; j < p.r; j += 8) {
        float v[8];
        load8_f32<TA>(b + j, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(t[j + e], v[e], s);
      }
    } else {
      for (int j = 0; j < p.r; ++j) s = fmaf(t[j], to_f32(b[j]), s);
    }
    s *= p.scale ? p.scale[ad] : 1.f;
  }
  out[row * p.d_out + n] = s;
}

// ------------------------------------------------------------------------------------------------ tiles
// Tile `i` of the rows: rows [row0, row0 + rows) of one group.
__device__ __forceinline__ void ad_tile(const AdaptArgs& p, int64_t i, int64_t& row0, int& rows) {
  const int64_t per = (p.rows_per_adapter + AD_TILE_ROWS - 1) / AD_TILE_ROWS;
  const int64_t group = i / per, in = (i - group * per) * AD_TILE_ROWS;
  row0 = group * p.rows_per_adapter + in;
  const int64_t end = min(min((group + 1) * p.rows_per_adapter, p.n_rows), row0 + AD_TILE_ROWS);
  rows = (int)max((int64_t)0, end - row0);
}

// A [rows x 32] block of a 16- or 32-bit matrix into shared memory as [32][ROWS + 4] floats (k outer), zeros outside.
// 8 threads a row of 32 values: 4 values each.
template <int ROWS, typename T>
__device__ __forceinline__ void ad_load(float (*dst)[ROWS + 4], const T* src, int64_t ld, int rows, int k0, int k1) {
  for (int i = threadIdx.x; i < ROWS * 8; i += 128) {
    const int r = i >> 3, k = (i & 7) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const T* s = src + r * ld + k0 + k;
      if (k0 + k + 4 <= k1 && (reinterpret_cast<uintptr_t>(s) & (4 * sizeof(T) - 1)) == 0) {
        if constexpr (sizeof(T) == 4) {
          const float4 f = *reinterpret_cast<const float4*>(s);
          v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(s);
          const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = to_f32(h[e]);
        }
      } else {
        for (int e = 0; e < 4; ++e) v[e] = k0 + k + e < k1 ? to_f32(s[e]) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) dst[k + e][r] = v[e];
  }
}

// t[z][row][j] over d_in split z: 64 rows x 32 ranks a CTA of 128 threads, 4 x 4 outputs each.
template <typename TX, typename TA>
__global__ void __launch_bounds__(128) adapt_shrink_tile_kernel(const TX* __restrict__ x, const AdaptArgs p) {
  __shared__ __align__(16) float xs[AD_BK][AD_TILE_ROWS + 4];
  __shared__ __align__(16) float as[AD_BK][AD_TILE_J + 4];
  pdl_trigger();
  pdl_wait();
  int64_t row0;
  int rows;
  ad_tile(p, blockIdx.x, row0, rows);
  if (rows <= 0) return;
  const int ad = ad_of(p, row0);
  if (ad < 0) return;
  const int j0 = blockIdx.y * AD_TILE_J, nj = min(AD_TILE_J, p.r - j0);
  const int steps = (p.d_in + AD_BK - 1) / AD_BK, per = (steps + p.splits - 1) / p.splits;
  const int kb = blockIdx.z * per * AD_BK, ke = min(p.d_in, kb + per * AD_BK);
  const TX* xr = x + row0 * p.d_in;
  const TA* ar = static_cast<const TA*>(p.a) + ((int64_t)ad * p.r + j0) * p.d_in;
  const int ty = threadIdx.x >> 3, tx = threadIdx.x & 7;  // 16 x 8 threads
  float acc[4][4] = {};
  for (int k0 = kb; k0 < ke; k0 += AD_BK) {
    ad_load<AD_TILE_ROWS, TX>(xs, xr, p.d_in, rows, k0, ke);
    ad_load<AD_TILE_J, TA>(as, ar, p.d_in, nj, k0, ke);
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < AD_BK; ++k) {
      const float4 u = *reinterpret_cast<const float4*>(&xs[k][ty * 4]);
      const float4 v = *reinterpret_cast<const float4*>(&as[k][tx * 4]);
      const float uu[4] = {u.x, u.y, u.z, u.w}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(uu[i], vv[j], acc[i][j]);
    }
    __syncthreads();
  }
  float* t = p.t + (int64_t)blockIdx.z * p.n_rows * p.r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (ty * 4 + i < rows && tx * 4 + j < nj) t[(row0 + ty * 4 + i) * p.r + j0 + tx * 4 + j] = acc[i][j];
}

// The same with mma.sync where x and A have one 16-bit type and 16-byte rows (products exact, sums in float32): a warp
// takes 16 rows x 32 ranks. The order of a dot product's terms is free, so lane l holds 8 consecutive columns of its rows
// (one 16-byte load from global memory, nothing staged) and the four lanes of a row make two k-steps of them. The tensor
// core's sums, which lose up to 2^-24 a step towards zero, are added up in float32 every 128 columns.
template <typename T>
__global__ void __launch_bounds__(128) adapt_shrink_mma_kernel(const T* __restrict__ x, const AdaptArgs p) {
  pdl_trigger();
  pdl_wait();
  int64_t row0;
  int rows;
  ad_tile(p, blockIdx.x, row0, rows);
  const int w0 = (threadIdx.x >> 5) * 16;  // this warp's first row of the tile
  if (rows <= w0) return;
  const int ad = ad_of(p, row0);
  if (ad < 0) return;
  const int lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const int j0 = blockIdx.y * AD_TILE_J, nj = min(AD_TILE_J, p.r - j0);
  const int steps = (p.d_in + AD_BK - 1) / AD_BK, per = (steps + p.splits - 1) / p.splits;
  const int kb = blockIdx.z * per * AD_BK, ke = min(p.d_in, kb + per * AD_BK);
  const bool in0 = w0 + r < rows, in1 = w0 + r + 8 < rows;
  const T* x0 = x + (row0 + w0 + r) * p.d_in + q * 8;
  const T* x1 = x0 + 8 * (int64_t)p.d_in;
  const T* ar = static_cast<const T*>(p.a) + ((int64_t)ad * p.r + j0 + r) * p.d_in + q * 8;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float sum[4][4] = {};
  for (int k0 = kb; k0 < ke; k0 += 4 * AD_BK) {
    float acc[4][4] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + u * AD_BK;
      const bool in = k + q * 8 < ke;  // (d_in is a multiple of 8, and so is every split's end)
      const uint4 a0 = in && in0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
      const uint4 a1 = in && in1 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 b = in && n * 8 + r < nj ? *reinterpret_cast<const uint4*>(ar + (int64_t)n * 8 * p.d_in + k) : zero;
        mma16816<T>(acc[n], a0.x, a1.x, a0.y, a1.y, b.x, b.y);
        mma16816<T>(acc[n], a0.z, a1.z, a0.w, a1.w, b.z, b.w);
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[n][e] += acc[n][e];
  }
  float* t = p.t + ((int64_t)blockIdx.z * p.n_rows + row0 + w0 + r) * p.r + j0;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = n * 8 + q * 2 + e;
      if (j >= nj) continue;
      if (in0) t[j] = sum[n][e];
      if (in1) t[8 * (int64_t)p.r + j] = sum[n][2 + e];
    }
}

// out[row][n] = s_a sum_j (sum_z t[z][row][j]) B[a][n][j]: 64 rows x 128 columns a CTA of 128 threads, 8 x 8 outputs.
template <typename TA>
__global__ void __launch_bounds__(128) adapt_expand_tile_kernel(const AdaptArgs p, float* __restrict__ out) {
  __shared__ __align__(16) float ts[AD_BK][AD_TILE_ROWS + 4];
  __shared__ __align__(16) float bs[AD_BK][AD_TILE_N + 4];
  pdl_trigger();
  pdl_wait();
  int64_t row0;
  int rows;
  ad_tile(p, blockIdx.x, row0, rows);
  if (rows <= 0) return;
  const int ad = ad_of(p, row0);
  const int n0 = blockIdx.y * AD_TILE_N, nn = min(AD_TILE_N, p.d_out - n0);
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;  // 8 x 16 threads
  float acc[8][8] = {};
  if (ad >= 0) {
    const TA* br = static_cast<const TA*>(p.b) + ((int64_t)ad * p.d_out + n0) * p.r;
    for (int k0 = 0; k0 < p.r; k0 += AD_BK) {
      for (int i = threadIdx.x; i < AD_TILE_ROWS * AD_BK; i += 128) {
        const int r = i / AD_BK, k = i % AD_BK;
        float v = 0.f;
        if (r < rows && k0 + k < p.r)
          for (int z = 0; z < p.splits; ++z) v += p.t[((int64_t)z * p.n_rows + row0 + r) * p.r + k0 + k];
        ts[k][r] = v;
      }
      ad_load<AD_TILE_N, TA>(bs, br, p.r, nn, k0, p.r);
      __syncthreads();
#pragma unroll 4
      for (int k = 0; k < min(AD_BK, p.r - k0); ++k) {
        float u[8], v[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          *reinterpret_cast<float4*>(u + 4 * h) = *reinterpret_cast<const float4*>(&ts[k][ty * 8 + 4 * h]);
          *reinterpret_cast<float4*>(v + 4 * h) = *reinterpret_cast<const float4*>(&bs[k][tx * 4 + 64 * h]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(u[i], v[j], acc[i][j]);
      }
      __syncthreads();
    }
  }
  const float c = ad >= 0 && p.scale ? p.scale[ad] : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (ty * 8 + i >= rows) break;
    float* o = out + (row0 + ty * 8 + i) * p.d_out + n0;
#pragma unroll
    for (int h = 0; h < 2; ++h)  // (d_out % 4 == 0)
      if (tx * 4 + 64 * h < nn)
        *reinterpret_cast<float4*>(o + tx * 4 + 64 * h) = make_float4(acc[i][4 * h] * c, acc[i][4 * h + 1] * c,
                                                                      acc[i][4 * h + 2] * c, acc[i][4 * h + 3] * c);
  }
}

}  // namespace xencb
