// Projection GEMM on 8-bit floating point operands (e4m3) with a power of two for each row's block of 128 columns, on the
// block-scaled tensor-core instructions (tcgen05.mma kind::mxf8f6f4), split-K.
//
//   x8[r, k] = rn_e4m3(x[r, k] 2^-ex[r, b]),  b = k / 128,  ex the smallest integer with max_b |x| <= 448 * 2^ex
//   part[z][m][n] = sum_{blocks b of split z} 2^(ex[m, b] + ew[n, b]) sum_{k in b} X8[m, k] W8[n, k]
//
// A power of two costs a floating-point format nothing but range, and the tensor core applies it itself (ue8m0 scale
// factors), so the accumulator runs over the whole split in float32. The instruction takes a scale per row and 32 columns:
// the four products of a block use the same one. The factors of a CTA's rows lie in tensor memory for all of its blocks,
// four blocks to a 32-bit word; the instruction descriptor names the byte.
//
// gemm_f8_kernel: D[n][m] (128 output features = UMMA M, BN rows of X = UMMA N). Warp 0 loads W8 and X8 tiles of 128 bytes
// a row by TMA into a ring, warp 1 issues four products a block, warps 2-5 bring the scale factors into tensor memory and
// store the split partial (a warp's lanes are consecutive columns). Values that are not finite become NaN, and so does
// every output of their row.
#pragma once

#include "gemm_f16x3.cuh"

namespace xencb {

constexpr int F8_BM = 128;   // output features per CTA
constexpr int F8_BK = 128;   // columns of a block: one scale factor a row, one 128-byte swizzle row
constexpr int F8_THREADS = 32 * 6;
__host__ __device__ constexpr int f8_stage(int bn) { return (F8_BM + bn) * F8_BK; }
__host__ __device__ constexpr int f8_stages(int bn) { return bn == 64 ? 8 : bn == 128 ? 6 : 4; }
__host__ __device__ constexpr size_t f8_smem(int bn) { return 1024 + (size_t)f8_stages(bn) * f8_stage(bn) + 256; }
// columns of tensor memory: BN of the accumulator, then per word of four blocks 4 of W's factors and BN / 32 of X's
__host__ __device__ constexpr int f8_word_cols(int bn) { return 4 + bn / 32; }
__host__ __device__ constexpr int f8_max_words(int bn) { return (512 - bn) / f8_word_cols(bn); }

// 2^e for e in [-127, 127]
__device__ __forceinline__ float f8_exp2i(int e) { return e > -127 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << 22); }

// ------------------------------------------------------------------------------------------------ to 8 bits
// One warp per (row, block): lane l holds columns 4 l .. 4 l + 3. x8 rows are kp = 128 ceil(K / 128) bytes, zeros behind
// column K; scale[row * stride + b] = e + 127.
template <typename T>
__device__ __forceinline__ void f8_load4(const T* __restrict__ row, int k, int K, bool vec, float* v) {
  if (vec && k + 4 <= K) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + k);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(row + k);
      T t[4];
      memcpy(t, &u, 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
  }
}

// The exponent of a block whose largest finite value is mx: mx = m 2^x with m in [1/2, 1), 448 = (7/8) 2^9.
__device__ __forceinline__ int f8_exponent(float mx) {
  if (!(mx > 0.f)) return 0;
  int x;
  const float m = frexpf(mx, &x);
  return max(-127, min(127, x - 9 + (m > 0.875f ? 1 : 0)));
}

// Four values as e4m3 bytes (round to nearest even); what is not finite as NaN.
__device__ __forceinline__ uint32_t f8_pack4(const float* v, float s) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * s), "f"(v[0] * s));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * s), "f"(v[2] * s));
  uint32_t u = (uint32_t)lo | ((uint32_t)hi << 16);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (!isfinite(v[i])) u |= 0x7fu << (8 * i);
  return u;
}

constexpr int F8Q_WARPS = 8;

template <typename T>
__global__ void __launch_bounds__(32 * F8Q_WARPS) quant_f8_kernel(const T* __restrict__ x, int64_t M, int K, int vec,
                                                                  uint8_t* __restrict__ x8,
                                                                  uint8_t* __restrict__ scale, int stride) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int nb = (K + F8_BK - 1) / F8_BK;
  const int64_t n = M * nb, step = (int64_t)gridDim.x * F8Q_WARPS;
  for (int64_t i = (int64_t)blockIdx.x * F8Q_WARPS + (threadIdx.x >> 5); i < n; i += step) {
    const int64_t m = i / nb;
    const int b = (int)(i - m * nb);
    float v[4];
    f8_load4<T>(x + m * K, b * F8_BK + lane * 4, K, vec, v);
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = fmaxf(mx, isfinite(v[j]) ? fabsf(v[j]) : 0.f);
    const int e = f8_exponent(warp_max(mx));
    const uint32_t u = f8_pack4(v, f8_exp2i(-e));
    reinterpret_cast<uint32_t*>(x8 + (m * nb + b) * F8_BK)[lane] = u;
    if (lane == 0) scale[m * stride + b] = (uint8_t)(e + 127);
  }
}

// ------------------------------------------------------------------------------------------------ product
// Instruction descriptor of the block-scaled kinds: [4,6) byte of B's scale word | [7,10) A format | [10,13) B format
// (0 e4m3) | [17,23) N >> 3 | 23 scale type (1 = ue8m0) | [27,29) M >> 7 | [29,31) byte of A's scale word.
__host__ __device__ constexpr uint32_t f8_idesc(int N, int byte) {
  return ((uint32_t)byte << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | (1u << 27) | ((uint32_t)byte << 29);
}

// D[tmem] (+)= (A 2^sa)(B 2^sb)^T over 32 columns, issued by one thread; sa, sb: the tensor-memory columns of the rows'
// scale words.
__device__ __forceinline__ void tc_mma_mx8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sa,
                                           uint32_t sb, bool acc) {
  const uint32_t en = acc ? 1u : 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(en)
      : "memory");
}

// 32 lanes x 1 column
__device__ __forceinline__ void tc_st1(uint32_t taddr, uint32_t v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(v) : "memory");
}

// Scale bytes of blocks 4 w .. 4 w + 3 of a row (1 behind the last).
__device__ __forceinline__ uint32_t f8_scale_word(const uint8_t* __restrict__ s, int nb, int w) {
  uint32_t u = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) u |= (w * 4 + i < nb ? (uint32_t)s[w * 4 + i] : 127u) << (8 * i);
  return u;
}

struct F8Args {
  int64_t M;
  int N, nb, bps;  // blocks of K, blocks per split
  const uint8_t* sw;  // [N, nb]
  const uint8_t* sx;  // [M, sx_stride]
  int sx_stride;
  float* part;
  int* row_done;
};

template <int BN>
__global__ void __launch_bounds__(F8_THREADS, 1) gemm_f8_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                const __grid_constant__ CUtensorMap map_x,
                                                                const F8Args a) {
  constexpr int STAGES = f8_stages(BN), STAGE = f8_stage(BN);
  extern __shared__ unsigned char f8_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* sfree = full + STAGES;
  uint64_t* done = sfree + STAGES;
  uint64_t* sf_ready = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * F8_BM;
  const int64_t m0 = (int64_t)blockIdx.y * BN;
  const int b0 = blockIdx.z * a.bps, b1 = min(a.nb, b0 + a.bps);
  const int nkb = max(0, b1 - b0), w0 = b0 / 4;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&sfree[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(sf_ready, 4);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tc_alloc(tmem_slot, 512);
    tc_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t taddr = *tmem_slot;
  // one stage of weights before the wait, as the 3xF16 GEMM does
  const int npre = min(nkb, 1);
  if (threadIdx.x != 0) {
    pdl_wait();
    pdl_trigger();
  }
  if (a.row_done && blockIdx.x == 0 && blockIdx.z == 0)
    for (int64_t i = m0 + threadIdx.x; i < min(a.M, m0 + BN); i += blockDim.x)
      if (threadIdx.x != 0) a.row_done[i] = 0;

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t keep = policy_evict_last();
      for (int kb = 0; kb < npre; ++kb) {
        mbar_arrive_expect_tx(&full[kb], STAGE);
        tma_load_2d_hint(smem + kb * STAGE, &map_w, (b0 + kb) * F8_BK, n0, &full[kb], keep);
      }
      pdl_wait();
      pdl_trigger();
      if (a.row_done && blockIdx.x == 0 && blockIdx.z == 0)
        for (int64_t i = m0; i < min(a.M, m0 + BN); i += blockDim.x) a.row_done[i] = 0;
      uint32_t used = 0;
      for (int kb = 0; kb < nkb; ++kb) {
        const int s = kb % STAGES, use = kb / STAGES;
        if (use > 0 && (!mbar_wait_spin(&sfree[s], (use - 1) & 1) || *abort_flag)) { *abort_flag = 1; break; }
        unsigned char* st = smem + s * STAGE;
        if (kb >= npre) {
          mbar_arrive_expect_tx(&full[s], STAGE);
          tma_load_2d_hint(st, &map_w, (b0 + kb) * F8_BK, n0, &full[s], keep);
        }
        tma_load_2d(st + F8_BM * F8_BK, &map_x, (b0 + kb) * F8_BK, (int)m0, &full[s]);
        used = kb + 1;
      }
      // after a wait that ran out: the copies in flight end before the CTA's shared memory goes away
      if (*abort_flag)
        for (uint32_t kb = used > STAGES ? used - STAGES : 0; kb < used; ++kb)
          mbar_wait_bounded(&full[kb % STAGES], (kb / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = nkb > 0 && mbar_wait_spin(sf_ready, 0);
      tc_fence_after();
      for (int kb = 0; kb < nkb && ok; ++kb) {
        const int s = kb % STAGES;
        if (!mbar_wait_spin(&full[s], (kb / STAGES) & 1) || *abort_flag) { ok = false; break; }
        tc_fence_after();
        const uint32_t sb = smem_u32(smem + s * STAGE);
        const int b = b0 + kb, word = b / 4 - w0;
        const uint32_t sa = taddr + BN + word * f8_word_cols(BN);
        const uint32_t idesc = f8_idesc(BN, 0) | ((uint32_t)(b & 3) << 4) | ((uint32_t)(b & 3) << 29);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)  // 32 columns: 32 bytes along the swizzle row
          tc_mma_mx8(taddr, umma_desc_k_sw128(sb + ks * 32), umma_desc_k_sw128(sb + F8_BM * F8_BK + ks * 32), idesc, sa,
                     sa + 4, kb > 0 || ks > 0);
        tc_commit(&sfree[s]);
      }
      if (!ok) *abort_flag = 1;
      tc_commit(done);
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter of this warp
    const uint32_t tl = taddr + ((uint32_t)(q * 32) << 16);
    // scale words: row 32 j + lane in column j, the same in every lane quarter
    const int words = nkb > 0 ? (b1 - 1) / 4 - w0 + 1 : 0;
    for (int w = 0; w < words; ++w) {
      uint32_t u[f8_word_cols(BN)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + j * 32 + lane;
        u[j] = n < a.N ? f8_scale_word(a.sw + (int64_t)n * a.nb, a.nb, w0 + w) : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int j = 0; j < BN / 32; ++j) {
        const int64_t m = m0 + j * 32 + lane;
        u[4 + j] = m < a.M ? f8_scale_word(a.sx + m * a.sx_stride, a.nb, w0 + w) : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int j = 0; j < f8_word_cols(BN); ++j) tc_st1(tl + BN + w * f8_word_cols(BN) + j, u[j]);
    }
    tc_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(sf_ready);
    const int n = n0 + q * 32 + lane;
    float* out = a.part + (int64_t)blockIdx.z * a.M * a.N;
    const int rows = (int)min((int64_t)BN, a.M - m0);
    const bool ok = nkb > 0 && mbar_wait_bounded(done, 0) && !*abort_flag;
    __syncwarp();
    tc_fence_after();
    for (int c = 0; c < rows; c += 32) {
      float v[32];
      tc_ld32(tl + (uint32_t)c, v);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c + i < rows && n < a.N) out[(m0 + c + i) * a.N + n] = ok ? v[i] : 0.f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_dealloc(taddr, 512);
  }
}

}  // namespace xencb
