// Projection GEMM on 8-bit floating point operands (e4m3) with a power of two for each row's block of 128 columns, on the
// block-scaled tensor-core instructions (tcgen05.mma kind::mxf8f6f4), split-K.
//
//   x8[r, k] = rn_e4m3(x[r, k] 2^-ex[r, b]),  b = k / 128,  ex the smallest integer with max_b |x| <= 448 * 2^ex
//   part[z][m][n] = sum_{blocks b of split z} 2^(ex[m, b] + ew[n, b]) sum_{k in b} X8[m, k] W8[n, k]
//
// A power of two costs a floating-point format nothing but range, and the tensor core applies it itself (ue8m0 scale
// factors), so the accumulator runs over a split's blocks in float32. The instruction takes a scale per row and 32 columns:
// the four products of a block use the same one. The factors of a CTA's rows lie in tensor memory for all of its blocks,
// four blocks to a 32-bit word; the instruction descriptor names the byte.
//
// gemm_f8_kernel: D[n][m] (128 output features = UMMA M, BN rows of X = UMMA N). Warp 0 loads W8 and X8 tiles of 128 bytes
// a row by TMA into a ring, warp 1 issues four products a block, warps 2-5 bring the scale factors into tensor memory and
// store the split partial (a warp's lanes are consecutive columns). Up to 8 rows warps 2-5 bring X's tiles into 8 bits
// themselves (TX its type; every band of 128 features does it again), a launch less: one token 4096 -> 2048 18.7 us a call in
// place of 21.4 (9.6 captured either way); 64 rows took 21 us captured that way against 9.9, so more rows are quantised
// by a launch of their own. Values that are not finite become NaN, and so does every output of their row.
//
// What bounds it: 64 rows 4096 -> 2048 (8.9 MB) take 6.8 us a launch, latency of the ring's first tiles and the split
// partials; the operands of many rows are gemm_f8_rows_kernel's, below.
#pragma once

#include "project.cuh"
#include "read_shared.cuh"

namespace xencb {

constexpr int F8_BM = 128;   // output features per CTA
constexpr int F8_BK = 128;   // columns of a block: one scale factor a row, one 128-byte swizzle row
constexpr int F8_THREADS = 32 * 6;
// Blocks that one accumulator runs over. The tensor core's drops bits below its running value at every product, towards zero:
// 3.5e-8 to 4.4e-8 of the result for each block (32, 40, 64 and 94 blocks: 1.1e-6, 1.6e-6, 2.8e-6 and 4.1e-6 off in norm;
// float32 sums are 2e-7 to 4e-7 off). Longer splits are cut; the rows kernel, below, takes its accumulator out more often.
constexpr int F8_RUN = 20;
__host__ __device__ constexpr int f8_stage(int bn) { return (F8_BM + bn) * F8_BK; }
__host__ __device__ constexpr int f8_stages(int bn) { return bn == 64 ? 8 : bn == 128 ? 6 : 4; }
__host__ __device__ constexpr size_t f8_smem(int bn) { return 1024 + (size_t)f8_stages(bn) * f8_stage(bn) + 1024; }
// columns of tensor memory: BN of the accumulator, then per word of four blocks 4 of W's factors and BN / 32 of X's
__host__ __device__ constexpr int f8_word_cols(int bn) { return 4 + bn / 32; }
__host__ __device__ constexpr int f8_max_words(int bn) { return (512 - bn) / f8_word_cols(bn); }

// 2^e for e in [-127, 127]
__device__ __forceinline__ float f8_exp2i(int e) { return e > -127 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << 22); }

// ------------------------------------------------------------------------------------------------ to 8 bits
// 8 values of a row from column k on (zeros behind column K); vec: 16-byte aligned rows of a multiple of 8 columns.
template <typename T>
__device__ __forceinline__ void f8_load8(const T* __restrict__ row, int k, int K, bool vec, float* v) {
  if (vec && k < K) {
    load8_f32<T>(row + k, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
  }
}

// The exponent of a block whose largest value has the bits mx (finite): mx = m 2^x with m in [1/2, 1), 448 = (7/8) 2^9.
// Values below 2^-126 have x <= -126: they get the smallest exponent.
__device__ __forceinline__ int f8_exponent(uint32_t mx) {
  if (mx == 0u) return 0;
  return max(-127, min(127, (int)(mx >> 23) - 126 - 9 + ((mx & 0x7fffffu) > 0x600000u ? 1 : 0)));
}

__device__ __forceinline__ uint32_t f8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four values as e4m3 bytes (round to nearest even).
__device__ __forceinline__ uint32_t f8_pack4(const float* v, float s) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1] * s), "f"(v[0] * s));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3] * s), "f"(v[2] * s));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// 8 consecutive values of a lane as e4m3 bytes, and the exponent of their block, which 16 consecutive lanes hold (all 32
// take part; `in`: this lane has values).
__device__ __forceinline__ uint2 f8_quant8(const float* v, bool in, int* e) {
  uint32_t mx = 0u;
  if (in) {
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = max(mx, f8_bits(v[j]));
  }
  uint32_t top = mx;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool odd = __any_sync(0xffffffffu, mx >= 0x7f800000u);  // a value of the warp that is not finite
  if (odd) {  // the largest finite one decides
    top = 0u;
    if (in) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, f8_bits(v[j]) < 0x7f800000u ? f8_bits(v[j]) : 0u);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  uint2 p = make_uint2(0u, 0u);
  *e = f8_exponent(top);
  if (!in) return p;
  const float s = f8_exp2i(-*e);
  p.x = f8_pack4(v, s);
  p.y = f8_pack4(v + 4, s);
  if (odd) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (f8_bits(v[j]) >= 0x7f800000u) (j < 4 ? p.x : p.y) |= 0x7fu << (8 * (j & 3));
  }
  return p;
}

// What the projection takes of a row besides its 8-bit form (project_in): 1/rms and the gate.
struct F8RowStats {
  int rms;
  float eps;
  const float* gate_w;  // [K] or null
  float gate_b;
  const float* gate_b_dev;
  float* rstd;          // [M]; null: no statistics
  float* gate;          // [M] or null
};

// HBM bounds it: 16384 float32 rows of 2048 (168 MB with their 8-bit form) take 28 us, 6.0 TB/s. 128 threads a row of float32
// (256: 38 us), 256 of 16 bits (2048 rows of 5120 7.6 us, with 128 7.9; 16384 rows of 4096 43, with 128 37).
// One CTA per row, 16 threads a block of 128 columns (8 values each, four times as many of a thread on their way, held as
// they came). x8 rows are kp = 128 ceil(K / 128) bytes, zeros behind column K; scale[row * stride + b] = e + 127.
template <typename T> __host__ __device__ constexpr int f8q_threads() { return sizeof(T) == 4 ? 128 : 256; }

// 8 values as they lie in memory.
template <typename T> struct F8Raw {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* __restrict__ row, int k, int K, bool vec) {
    if (vec && k < K) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(row + k)[i];
    } else {
      T t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = k + i < K ? row[k + i] : from_f32<T>(0.f);
      memcpy(u, t, sizeof(t));
    }
  }
  __device__ __forceinline__ void values(float* v) const {
    if constexpr (sizeof(T) == 4) {
      unpack16<T>(u[0], v);
      unpack16<T>(u[1], v + 4);
    } else {
      unpack16<T>(u[0], v);
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(f8q_threads<T>(), sizeof(T) == 4 ? 8 : 6) quant_f8_kernel(const T* __restrict__ x, int K, int vec,
                                                               uint8_t* __restrict__ x8, uint8_t* __restrict__ scale,
                                                               int stride, const F8RowStats st) {
  __shared__ float2 red[32];
  pdl_trigger();
  pdl_wait();
  const int64_t m = blockIdx.x;
  const T* row = x + m * K;
  const int kp = (K + F8_BK - 1) / F8_BK * F8_BK;
  float ss = 0.f, gd = 0.f;
  constexpr int U = 4, STEP = f8q_threads<T>() * 8;
  for (int k0 = 0; k0 < kp; k0 += STEP * U) {
    F8Raw<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * STEP + (int)threadIdx.x * 8;
      if (k < kp) raw[u].load(row, k, K, vec);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * STEP + (int)threadIdx.x * 8;
      if (k0 + u * STEP >= kp) break;
      float v[8];
      raw[u].values(v);
      int e;
      const uint2 p = f8_quant8(v, k < kp, &e);
      if (k >= kp) continue;
      *reinterpret_cast<uint2*>(x8 + m * kp + k) = p;
      if ((threadIdx.x & 15) == 0) scale[m * stride + k / F8_BK] = (uint8_t)(e + 127);
      if (st.rstd) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        if (st.gate_w) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k + j < K) gd = fmaf(v[j], __ldg(st.gate_w + k + j), gd);
        }
      }
    }
  }
  if (!st.rstd) return;
  const float2 t = block_sum2(ss, gd, red);
  if (threadIdx.x == 0) {
    const float rstd = st.rms ? rsqrtf(t.x / (float)K + st.eps) : 1.f;
    st.rstd[m] = rstd;
    if (st.gate) {
      const float gb = st.gate_b_dev ? __ldg(st.gate_b_dev) : st.gate_b;
      st.gate[m] = 1.f / (1.f + expf(-(t.y * rstd + gb)));
    }
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

// Scale bytes of blocks 4 w .. 4 w + 3 of a row (1 behind the last); words: the row is a whole number of aligned words.
__device__ __forceinline__ uint32_t f8_scale_word(const uint8_t* __restrict__ s, int nb, int w, bool words) {
  if (words) return __ldg(reinterpret_cast<const uint32_t*>(s) + w);
  uint32_t u = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) u |= (w * 4 + i < nb ? (uint32_t)s[w * 4 + i] : 127u) << (8 * i);
  return u;
}

struct F8Args {
  int64_t M;
  int N, nb, bps;  // blocks of K, blocks per split
  const uint8_t* sw;  // [N, nb]
  const uint8_t* sx;  // [M, sx_stride], rows of aligned words
  int sx_stride;
  int sw_words;       // W's rows too
  float* part;
  int* row_done;
  const void* x;  // TX [M, K]: the rows as they are
  int K, vec;
};

// X's factors lie behind W's: a word of four blocks like W's, or (TX) a word of one block, in BN / 32 columns.
constexpr int F8_FUSED_ROWS = 8;

template <int BN, typename TX>
__global__ void __launch_bounds__(F8_THREADS, 1) gemm_f8_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                const __grid_constant__ CUtensorMap map_x,
                                                                const F8Args a) {
  constexpr int STAGES = f8_stages(BN), STAGE = f8_stage(BN);
  constexpr bool FUSED = !std::is_void<TX>::value;
  static_assert(!FUSED || BN == 64, "two columns of X's factors a block");
  constexpr int WCOLS = FUSED ? 4 : f8_word_cols(BN);
  __shared__ uint8_t xs_sh[FUSED ? 8 * F8_FUSED_ROWS : 1];
  extern __shared__ unsigned char f8_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
  uint64_t* sfree = full + STAGES;
  uint64_t* done = sfree + STAGES;
  uint64_t* sf_ready = done + 1;  // one per word of scale factors
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_ready + f8_max_words(BN));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * F8_BM;
  const int64_t m0 = (int64_t)blockIdx.y * BN;
  const int b0 = blockIdx.z * a.bps, b1 = min(a.nb, b0 + a.bps);
  const int nkb = max(0, b1 - b0), w0 = b0 / 4;
  const int words = nkb > 0 ? (b1 - 1) / 4 - w0 + 1 : 0;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], FUSED ? 5 : 1);
      mbar_init(&sfree[i], 1);
    }
    mbar_init(done, 1);
    for (int i = 0; i < f8_max_words(BN); ++i) mbar_init(&sf_ready[i], 4);
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
  const uint64_t keep = policy_evict_last();
  // The first weights are asked into L2 before the wait, and read behind it: what wrote them (xencb_quant8, a copy) may be
  // the launch before this one.
  if (threadIdx.x == 0 && nkb > 0) tma_prefetch_2d(&map_w, b0 * F8_BK, n0, keep);
  pdl_wait();
  pdl_trigger();
  if (a.row_done && blockIdx.x == 0 && blockIdx.z == 0)
    for (int64_t i = m0 + threadIdx.x; i < min(a.M, m0 + BN); i += blockDim.x) a.row_done[i] = 0;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t used = 0;
      for (int kb = 0; kb < nkb; ++kb) {
        const int s = kb % STAGES, use = kb / STAGES;
        if (use > 0 && (!mbar_wait_spin(&sfree[s], (use - 1) & 1) || *abort_flag)) { *abort_flag = 1; break; }
        unsigned char* st = smem + s * STAGE;
        mbar_arrive_expect_tx(&full[s], FUSED ? F8_BM * F8_BK : STAGE);
        tma_load_2d_hint(st, &map_w, (b0 + kb) * F8_BK, n0, &full[s], keep);
        if (!FUSED) tma_load_2d(st + F8_BM * F8_BK, &map_x, (b0 + kb) * F8_BK, (int)m0, &full[s]);
        used = kb + 1;
      }
      // after a wait that ran out: the copies in flight end before the CTA's shared memory goes away
      if (*abort_flag)
        for (uint32_t kb = used > STAGES ? used - STAGES : 0; kb < used; ++kb)
          mbar_wait_bounded(&full[kb % STAGES], (kb / STAGES) & 1);
    }
  } else if (warp == 1) {
    if (elect_one()) {
      bool ok = nkb > 0;
      int ready = -1;
      for (int kb = 0; kb < nkb && ok; ++kb) {
        const int s = kb % STAGES;
        if ((b0 + kb) / 4 - w0 != ready) {
          ready = (b0 + kb) / 4 - w0;
          if (!(ok = mbar_wait_spin(&sf_ready[ready], 0))) break;
        }
        if (!mbar_wait_spin(&full[s], (kb / STAGES) & 1) || *abort_flag) { ok = false; break; }
        tc_fence_after();
        const uint32_t sb = smem_u32(smem + s * STAGE);
        const int b = b0 + kb, word = b / 4 - w0;
        if (FUSED) fence_proxy_async_smem();  // X's tile was written by this CTA's threads
        const uint32_t sa = taddr + BN + word * WCOLS;
        const uint32_t sx = FUSED ? taddr + BN + words * WCOLS + kb * (BN / 32) : sa + 4;
        const uint32_t idesc = f8_idesc(BN, 0) | (FUSED ? 0u : (uint32_t)(b & 3) << 4) | ((uint32_t)(b & 3) << 29);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)  // 32 columns: 32 bytes along the swizzle row
          tc_mma_mx8(taddr, umma_desc_k_sw128(sb + ks * 32), umma_desc_k_sw128(sb + F8_BM * F8_BK + ks * 32), idesc, sa,
                     sx, kb > 0 || ks > 0);
        tc_commit(&sfree[s]);
      }
      if (!ok) *abort_flag = 1;
      tc_commit(done);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;  // TMEM lane quarter of this warp
    const uint32_t tl = taddr + ((uint32_t)(q * 32) << 16);
    const int rows = (int)min((int64_t)BN, a.M - m0);
    // FUSED: thread t holds 8 values of row t / 16 in each of 8 blocks; the first are on their way before W's factors
    const int t = threadIdx.x - 64, xr = t >> 4, xk = (t & 15) * 8;
    float v[FUSED ? 8 : 1][8];
    auto load = [&](int kb) {
      if constexpr (FUSED) {
        const TX* x = static_cast<const TX*>(a.x) + (m0 + xr) * a.K;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
          if (xr < rows && kb + i < nkb) f8_load8<TX>(x, (b0 + kb + i) * F8_BK + xk, a.K, a.vec, v[i]);
        }
      }
    };
    if (FUSED && nkb > 0) load(0);
    // scale words: row 32 j + lane in column j, the same in every lane quarter
    for (int w = 0; w < words; ++w) {
      uint32_t u[WCOLS];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + j * 32 + lane;
        u[j] = n < a.N ? f8_scale_word(a.sw + (int64_t)n * a.nb, a.nb, w0 + w, a.sw_words) : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int j = 0; j < WCOLS - 4; ++j) {
        const int64_t m = m0 + j * 32 + lane;
        u[4 + j] = m < a.M ? f8_scale_word(a.sx + m * a.sx_stride, a.nb, w0 + w, true) : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int j = 0; j < WCOLS; ++j) tc_st1(tl + BN + w * WCOLS + j, u[j]);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_ready[w]);
      __syncwarp();
    }
    if constexpr (FUSED) {
      static_assert(!FUSED || STAGES == 8, "a round of 8 blocks fills the ring");
      for (int kb = 0; kb < nkb; kb += 8) {
        const int n = min(8, nkb - kb);
        if (kb > 0) {
          for (int i = 0; i < n; ++i)
            if (!*abort_flag && !mbar_wait_spin(&sfree[i], (kb / 8 - 1) & 1)) *abort_flag = 1;
          __syncwarp();
        }
        // (the eight blocks' reductions side by side)
        uint32_t top[8], any = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          top[i] = 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) top[i] = max(top[i], f8_bits(v[i][j]));
          any = max(any, top[i]);
        }
        const bool odd = __any_sync(0xffffffffu, any >= 0x7f800000u);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
#pragma unroll
          for (int i = 0; i < 8; ++i) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // 16-byte chunk c of row r at chunk c ^ (r % 8)
          int e = f8_exponent(top[i]);
          uint2 p;
          if (odd) {
            p = f8_quant8(v[i], true, &e);
          } else {
            const float sc = f8_exp2i(-e);
            p = make_uint2(f8_pack4(v[i], sc), f8_pack4(v[i] + 4, sc));
          }
          if (xr < rows && i < n) {
            unsigned char* tile = smem + i * STAGE + F8_BM * F8_BK;
            *reinterpret_cast<uint2*>(tile + xr * F8_BK + (((xk >> 4) ^ xr) << 4) + (xk & 8)) = p;
            if ((t & 15) == 0) xs_sh[i * F8_FUSED_ROWS + xr] = (uint8_t)(e + 127);
          }
        }
        if (kb + 8 < nkb) load(kb + 8);
        fence_proxy_async_smem();
        named_bar_sync(1, 128);
        for (int i = 0; i < n; ++i) {
          const uint32_t at = tl + BN + words * WCOLS + (kb + i) * (BN / 32);
          tc_st1(at, lane < rows ? xs_sh[i * F8_FUSED_ROWS + lane] : 127u);
          tc_st1(at + 1, 127u);
        }
        tc_wait_st();
        tc_fence_before();
        named_bar_sync(1, 128);  // (every warp has read the bytes; the next round writes them)
        if (lane == 0)
          for (int i = 0; i < n; ++i) mbar_arrive(&full[i]);
        __syncwarp();
      }
    }
    const int n = n0 + q * 32 + lane;
    float* out = a.part + (int64_t)blockIdx.z * a.M * a.N;
    const bool ok = nkb > 0 && mbar_wait_bounded(done, 0) && !*abort_flag;
    __syncwarp();
    tc_fence_after();
    for (int c = 0; c < rows; c += 32) {
      float y[32];
      tc_ld32(tl + (uint32_t)c, y);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (c + i < rows && n < a.N) out[(m0 + c + i) * a.N + n] = ok ? y[i] : 0.f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_dealloc(taddr, 512);
  }
}

// ------------------------------------------------------------------------------------------------ many rows
// The same product with the rows of X as the 128-row operand and 256 output features as N, for calls that fill the device
// with such tiles: a thread of the epilogue holds 128 outputs of one row, so the projection's elementwise end is done
// where the product is and no partials are written. Persistent: 8 epilogue warps take the accumulator into registers and
// give it back before they store, so that the next tile's products run meanwhile; they also bring the next tile's scale
// factors (two sets of them in tensor memory).
// 16384 rows 2048 -> 4096 take 116 to 122 us, 2.3 PFLOP/s, with h + delta in place of delta 149, with the sums of the mag term
// too, as the hook calls it, 190 (h is loaded where it is used, beside v's 128 registers); 103 without the stores, 94 without
// the epilogue, 83 as the products alone: the operands (1.6 GB from L2), what the epilogue writes and its arithmetic each add
// about 11 to the products, which run at 3.3 PFLOP/s. (h on its way four groups before its use: 158.) 2048 rows 5120 -> 2048
// are one tile a CTA: 28 to 30 us, 15 of it products. The accumulator is taken out every FR_RUN blocks: 40 blocks at once were
// 1.6e-6 of the result off, in three runs 5e-7, for 1.3 us.
//   project_in   q = y * rstd + b; the row's sum of squares by pieces of 128 columns, for f8_norm_kernel
//   project_out  delta = scale * gate * (y + b) * mask in h's type, h + delta; sums of squares of delta and h for the mag term
constexpr int FR_BM = 128, FR_BN = 256, FR_STAGES = 4;
constexpr int FR_STAGE = (FR_BM + FR_BN) * F8_BK;
constexpr int FR_WORD_COLS = FR_BM / 32 + FR_BN / 32;
constexpr int FR_MAX_WORDS = (512 - FR_BN) / 2 / FR_WORD_COLS;  // two sets
constexpr int FR_RUN = 16;  // blocks that the accumulator runs over before it is added up in registers
constexpr int FR_EPI = 8;
constexpr int FR_THREADS = 32 * (4 + FR_EPI);
constexpr size_t FR_SMEM = 1024 + (size_t)FR_STAGES * FR_STAGE + 256;
constexpr int FR_REGS_LOW = 88, FR_REGS_HIGH = 208;
constexpr int FR_REGS = 4 * 32 * FR_REGS_LOW + 32 * FR_EPI * FR_REGS_HIGH;

struct F8RowsArgs {
  int64_t M;
  int N, nb, tiles_n;
  int64_t tiles;
  const uint8_t* sw;
  int sw_words;
  const uint8_t* sx;
  int sx_stride;
  const float* mul;   // [M]: 1/rms, or the gate; null: 1
  const float* bias;  // [N] or null
  float scale;        // project_out
  const float* log_scale_dev;
  const float* pos_mask;
  const void* h;      // [M, N] for out2
  void* out;          // q, or delta (or null)
  void* out2;         // h + delta, or null
  float2* sums;       // [M, 2 tiles_n]: sums of squares of q, or of (delta, h); null: none
  int vec;            // 32-byte stores: N and the bases allow them
};

// 32 bytes of a thread
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* u) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]),
               "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
__device__ __forceinline__ void ld_global_32(const void* p, uint32_t* u) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "l"(p));
}

template <typename TO, bool OUT>
__global__ void __launch_bounds__(FR_THREADS, 1) gemm_f8_rows_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                     const __grid_constant__ CUtensorMap map_w,
                                                                     const F8RowsArgs a) {
  extern __shared__ unsigned char fr_smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(fr_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + FR_STAGES * FR_STAGE);
  uint64_t* empty = full + FR_STAGES;
  uint64_t* acc_full = empty + FR_STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* sf_full = acc_empty + 1;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_full + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int words = (a.nb + 3) / 4;
  // the accumulator's runs, of nearly one length
  const int runs = (a.nb + FR_RUN - 1) / FR_RUN, run = (a.nb + runs - 1) / runs;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    for (int i = 0; i < FR_STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, FR_EPI);
    mbar_init(&sf_full[0], FR_EPI);
    mbar_init(&sf_full[1], FR_EPI);
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
  pdl_wait();
  pdl_trigger();

  if (warp < 4) {
    regs_dec<FR_REGS_LOW>();
    if (warp == 0) {
      if (elect_one()) {
        const uint64_t keep = policy_evict_last();
        RsRing ring{0, 0};
        uint32_t used = 0;
        bool ok = true;
        for (int64_t t = blockIdx.x; t < a.tiles && ok; t += gridDim.x) {
          const int m0 = (int)(t / a.tiles_n) * FR_BM, n0 = (int)(t % a.tiles_n) * FR_BN;
          for (int kb = 0; kb < a.nb; ++kb) {
            if (used >= FR_STAGES && !(ok = mbar_wait_spin(&empty[ring.st], ring.phase ^ 1))) break;
            unsigned char* st = smem + ring.st * FR_STAGE;
            mbar_arrive_expect_tx(&full[ring.st], FR_STAGE);
            tma_load_2d(st, &map_x, kb * F8_BK, m0, &full[ring.st]);
            tma_load_2d_hint(st + FR_BM * F8_BK, &map_w, kb * F8_BK, n0, &full[ring.st], keep);
            ring.next(FR_STAGES);
            ++used;
          }
        }
        if (!ok) {  // the copies in flight end before the CTA's shared memory goes away
          *abort_flag = 1;
          for (uint32_t i = min(used, (uint32_t)FR_STAGES); i > 0; --i) {
            ring.back(FR_STAGES);
            mbar_wait_bounded(&full[ring.st], ring.phase);
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      if (elect_one()) {
        RsRing ring{0, 0};
        bool ok = true;
        uint32_t i = 0, acc = 0;
        for (int64_t t = blockIdx.x; t < a.tiles && ok; t += gridDim.x, ++i) {
          if (!(ok = mbar_wait_spin(&sf_full[i & 1], (i >> 1) & 1))) break;
          const uint32_t sf = taddr + FR_BN + (i & 1) * (FR_MAX_WORDS * FR_WORD_COLS);
          for (int k0 = 0; k0 < a.nb && ok; k0 += run, ++acc) {
            if (acc > 0 && !(ok = mbar_wait_spin(acc_empty, (acc - 1) & 1))) break;
            tc_fence_after();
            const int k1 = min(a.nb, k0 + run);
            for (int kb = k0; kb < k1; ++kb) {
              if (!(ok = mbar_wait_spin(&full[ring.st], ring.phase))) break;
              tc_fence_after();
              const uint32_t sb = smem_u32(smem + ring.st * FR_STAGE);
              const uint32_t sa = sf + (kb >> 2) * FR_WORD_COLS;
              const uint32_t idesc = f8_idesc(FR_BN, 0) | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                tc_mma_mx8(taddr, umma_desc_k_sw128(sb + ks * 32), umma_desc_k_sw128(sb + FR_BM * F8_BK + ks * 32), idesc,
                           sa, sa + FR_BM / 32, kb > k0 || ks > 0);
              tc_commit(&empty[ring.st]);
              ring.next(FR_STAGES);
            }
            if (ok) tc_commit(acc_full);
          }
        }
        if (!ok) *abort_flag = 1;
      }
      __syncwarp();
    }
  } else {
    regs_inc<FR_REGS_HIGH>();
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t tl = taddr + ((uint32_t)(q * 32) << 16);
    auto done = [&](bool arrived) {
      if (!arrived) *abort_flag = 1;
      __syncwarp();
    };
    // the scale words of tile t: row 32 j + lane in column j, in every lane quarter; the two warps of a quarter take turns
    auto scales = [&](int64_t t, uint32_t i) {
      const int64_t m0 = t / a.tiles_n * FR_BM;
      const int n0 = (int)(t % a.tiles_n) * FR_BN;
      const uint32_t at = tl + FR_BN + (i & 1) * (FR_MAX_WORDS * FR_WORD_COLS);
      for (int w = half; w < words; w += 2) {
        uint32_t u[FR_WORD_COLS];
#pragma unroll
        for (int j = 0; j < FR_BM / 32; ++j) {
          const int64_t m = m0 + j * 32 + lane;
          u[j] = m < a.M ? f8_scale_word(a.sx + m * a.sx_stride, a.nb, w, true) : 0x7f7f7f7fu;
        }
#pragma unroll
        for (int j = 0; j < FR_BN / 32; ++j) {
          const int n = n0 + j * 32 + lane;
          u[FR_BM / 32 + j] = n < a.N ? f8_scale_word(a.sw + (int64_t)n * a.nb, a.nb, w, a.sw_words) : 0x7f7f7f7fu;
        }
#pragma unroll
        for (int j = 0; j < FR_WORD_COLS; ++j) tc_st1(at + w * FR_WORD_COLS + j, u[j]);
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sf_full[i & 1]);
      __syncwarp();
    };
    if (blockIdx.x < a.tiles) scales(blockIdx.x, 0);
    const float ls = a.log_scale_dev ? expf(__ldg(a.log_scale_dev)) : 1.f;
    uint32_t i = 0, acc = 0;
    for (int64_t t = blockIdx.x; t < a.tiles; t += gridDim.x, ++i) {
      // (the products of the tile before, which used this set, are done: its accumulator was waited for)
      if (t + gridDim.x < a.tiles) scales(t + gridDim.x, i + 1);
      const int64_t m = t / a.tiles_n * FR_BM + q * 32 + lane;
      const int n0 = (int)(t % a.tiles_n) * FR_BN + half * 128;
      const bool in = m < a.M;
      float mul = in && a.mul ? a.mul[m] : 1.f;
      if (OUT) mul *= a.scale * ls * (a.pos_mask && in ? a.pos_mask[m] : 1.f);
      auto arrived = [&] {
        done(*abort_flag || mbar_wait_spin(acc_full, acc & 1));
        tc_fence_after();
      };
      auto taken = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
        __syncwarp();
        ++acc;
      };
      float v[128];
      arrived();
#pragma unroll
      for (int g = 0; g < 128; g += 32) tc_ld32(tl + half * 128 + g, v + g);
      taken();
      for (int k0 = run; k0 < a.nb; k0 += run) {
        arrived();
#pragma unroll
        for (int g = 0; g < 128; g += 16) {  // (there are no registers for more beside v)
          float x[16];
          tc_ld16(tl + half * 128 + g, x);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[g + e] += x[e];
        }
        taken();
      }
      if (*abort_flag) {
#pragma unroll
        for (int g = 0; g < 128; ++g) v[g] = 0.f;
      }
      if (in) {
        TO* o = a.out ? static_cast<TO*>(a.out) + m * a.N + n0 : nullptr;
        TO* o2 = OUT && a.out2 ? static_cast<TO*>(a.out2) + m * a.N + n0 : nullptr;
        const TO* h = OUT && (a.out2 || a.sums) ? static_cast<const TO*>(a.h) + m * a.N + n0 : nullptr;
        constexpr int PER = 32 / sizeof(TO);  // values of a 32-byte store
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        // (one test a group for what a call has: a test for each value took the epilogue from 96 to 172 us, 16384 rows
        // 2048 -> 4096)
#pragma unroll
        for (int g = 0; g < 128; g += PER) {
          if (n0 + g >= a.N) break;
          const bool whole = n0 + g + PER <= a.N, vec = a.vec && whole;
          if (a.bias) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              const float b = whole || n0 + g + e < a.N ? __ldg(a.bias + n0 + g + e) : 0.f;
              v[g + e] = OUT ? mul * (v[g + e] + b) : fmaf(v[g + e], mul, b);
            }
          } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) v[g + e] *= mul;
          }
          alignas(32) TO x[PER], hx[PER];
#pragma unroll
          for (int e = 0; e < PER; ++e) x[e] = from_f32<TO>(v[g + e]);
          if (OUT && h) {
            if (vec) {
              ld_global_32(h + g, reinterpret_cast<uint32_t*>(hx));
            } else {
#pragma unroll
              for (int e = 0; e < PER; ++e) hx[e] = whole || n0 + g + e < a.N ? h[g + e] : from_f32<TO>(0.f);
            }
          }
          if (a.sums) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
              const float r = whole || n0 + g + e < a.N ? to_f32(x[e]) : 0.f;
              s0[e & 3] = fmaf(r, r, s0[e & 3]);
              if (OUT) {
                const float hv = to_f32(hx[e]);
                s1[e & 3] = fmaf(hv, hv, s1[e & 3]);
              }
            }
          }
          if (o) {
            if (vec) {
              st_global_32(o + g, reinterpret_cast<const uint32_t*>(x));
            } else {
#pragma unroll
              for (int e = 0; e < PER; ++e)
                if (whole || n0 + g + e < a.N) o[g + e] = x[e];
            }
          }
          if (OUT && o2) {
#pragma unroll
            for (int e = 0; e < PER; ++e) hx[e] = from_f32<TO>(to_f32(hx[e]) + to_f32(x[e]));
            if (vec) {
              st_global_32(o2 + g, reinterpret_cast<const uint32_t*>(hx));
            } else {
#pragma unroll
              for (int e = 0; e < PER; ++e)
                if (whole || n0 + g + e < a.N) o2[g + e] = hx[e];
            }
          }
        }
        if (a.sums) 
          a.sums[m * 2 * a.tiles_n + (t % a.tiles_n) * 2 + half] =
              make_float2((s0[0] + s0[1]) + (s0[2] + s0[3]), (s1[0] + s1[1]) + (s1[2] + s1[3]));
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tc_dealloc(taddr, 512);
}

// q /= ||q|| + 1e-6, one CTA per row.
__global__ void __launch_bounds__(256) f8_norm_kernel(float* __restrict__ q, int N, const float2* __restrict__ sums,
                                                      int n_sums) {
  pdl_trigger();
  pdl_wait();
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 31;
  float4* row = reinterpret_cast<float4*>(q + m * N);
  constexpr int HELD = 2;
  float4 v[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h)
    if (h * 256 + threadIdx.x < N / 4) v[h] = row[h * 256 + threadIdx.x];
  float t = 0.f;  // (every warp adds the pieces in the same order)
  for (int i = lane; i < n_sums; i += 32) t += sums[m * n_sums + i].x;
  const float den = sqrtf(warp_sum(t)) + 1e-6f;
#pragma unroll
  for (int h = 0; h < HELD; ++h)
    if (h * 256 + threadIdx.x < N / 4)
      row[h * 256 + threadIdx.x] = make_float4(v[h].x / den, v[h].y / den, v[h].z / den, v[h].w / den);
  for (int i = HELD * 256 + threadIdx.x; i < N / 4; i += 256) {
    const float4 w = row[i];
    row[i] = make_float4(w.x / den, w.y / den, w.z / den, w.w / den);
  }
}

// The mag term ||delta|| / (||h|| + 1e-6) of every row.
__global__ void __launch_bounds__(256) f8_rel_kernel(int64_t M, const float2* __restrict__ sums, int n_sums,
                                                     float* __restrict__ rel) {
  pdl_trigger();
  pdl_wait();
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= M) return;
  float d = 0.f, h = 0.f;
  for (int i = 0; i < n_sums; ++i) {
    const float2 t = sums[m * n_sums + i];
    d += t.x;
    h += t.y;
  }
  rel[m] = sqrtf(d) / (sqrtf(h) + 1e-6f);
}

}  // namespace xencb
