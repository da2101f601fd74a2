// Low-rank adapters beside the interface projections: y = x W^T + s_a (x A_a^T) B_a^T, where a = adapter_of[row /
// rows_per_adapter] (negative: none) picks one of n adapters A [n, r, d_in], B [n, d_out, r], s [n].
//
// The projection's row kernels sum split partials of the GEMM, so the low-rank term is one more partial: shrink
// t = x A_a^T, then expand s_a t B_a^T into the slice behind the GEMM's. It lies before 1/rms, the bias, the norms
// and the gate, as the GEMM's partials do, and is float32 throughout.
#pragma once

#include "common.cuh"

namespace xencb {

constexpr int AD_MAX_RANK = 256;

struct AdaptArgs {
  const void* a;        // [n, r, d_in]
  const void* b;        // [n, d_out, r]
  const float* scale;   // [n] or null (1)
  const int32_t* of;    // [ceil(n_rows / rows_per_adapter)]
  int64_t rows_per_adapter;
  int n, r, d_in, d_out;
  float* t;             // [n_rows, r]
};

// the adapter of a row, or -1; an index past the last adapter is flagged and read as none
__device__ __forceinline__ int ad_of(const AdaptArgs& p, int64_t row) {
  const int a = p.of[row / p.rows_per_adapter];
  if (a >= p.n) flag_error(XENCB_DEV_BADADAPTER);
  return a < 0 || a >= p.n ? -1 : a;
}

// t[row][j] = x[row] . A[a][j]: one CTA per row, one warp per j.
template <typename TX, typename TA>
__global__ void __launch_bounds__(256) adapt_shrink_kernel(const TX* __restrict__ x, const AdaptArgs p) {
  const int64_t row = blockIdx.x;
  const int ad = ad_of(p, row);
  if (ad < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int j = warp; j < p.r; j += 8) {
    const TA* a = static_cast<const TA*>(p.a) + ((int64_t)ad * p.r + j) * p.d_in;
    float s = 0.f;
    for (int k = lane; k < p.d_in; k += 32) s = fmaf(to_f32(x[row * p.d_in + k]), to_f32(a[k]), s);
    s = warp_sum(s);
    if (lane == 0) p.t[row * p.r + j] = s;
  }
}

// out[row][n] = s_a sum_j t[row][j] B[a][n][j]; 0 for a row without an adapter.
template <typename TA>
__global__ void __launch_bounds__(256) adapt_expand_kernel(const AdaptArgs p, float* __restrict__ out) {
  __shared__ float t[AD_MAX_RANK];
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
    for (int j = 0; j < p.r; ++j) s = fmaf(t[j], to_f32(b[j]), s);
    s *= p.scale ? p.scale[ad] : 1.f;
  }
  out[row * p.d_out + n] = s;
}

}  // namespace xencb
