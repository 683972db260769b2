// fp8 linears of a decoder layer: e4m3 values with power-of-two (e8m0) scales for blocks of 128.
//
//   scales   one byte s per block, standing for 2^(s - 127): a block is 128 consecutive values of a
//            row (activations, [rows][ceil(K/128)]) or 128 rows x 128 columns of a weight
//            ([ceil(N/128)][ceil(K/128)]); s = 255 stands for NaN, as the tensor cores read it.
//   quantise e = the least exponent >= -127 with max |v| <= 448 * 2^e over the block's finite values
//            (448 is the largest e4m3), q = e4m3(v * 2^-e) rounded to nearest even. Values that are not
//            finite become NaN and do not set the scale. 448 = 1.75 * 2^8, so e comes from the
//            maximum's exponent and one comparison of its fraction: no logarithm, no division.
//   norm     h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, then quantised as above, or to
//            int8 at a power-of-two position p: q = clamp(rne(y * 2^p), -128, 127), the activations of
//            the W4A8 and int8 products.
//   linear   out[m][n] = sum over blocks b of 2^(xs[m][b] + ws[n/128][b] - 254) * sum_{k in b} x[m][k] * w[n][k]
//   swiglu   g and u such products, y = g / (1 + exp(-g)) * u, quantised per 128 outputs of a row.
//
// Sums, norms and the epilogues are held in 32 bits; each output is rounded once.
#pragma once
#include <cfloat>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "ixb_gemm.cuh"
#include "ixb_ptx.cuh"

namespace ixb {

enum : int { FT_BF16 = 0, FT_F16 = 1, FT_F32 = 2 };  // IXB_BF16, IXB_F16, IXB_F32
constexpr int kQBlock = 128;                         // values that share a scale

// ---------------------------------------------------------------- conversions
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// Eight consecutive values, 16-byte aligned.
template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> r;
  const uint4* s = reinterpret_cast<const uint4*>(p);
  uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = s[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& r) {
  const uint4* s = reinterpret_cast<const uint4*>(&r);
  uint4* d = reinterpret_cast<uint4*>(p);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = s[i];
}

// |v| of a finite value, 0 of another one: what sets a block's scale.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= FLT_MAX ? a : 0.f;
}
// The scale byte of a block whose largest finite |v| is `top`: 448 * 2^(s - 127) >= top, s >= 0 least.
__device__ __forceinline__ uint32_t scale_byte(float top) {
  const uint32_t u = __float_as_uint(top);
  const int s = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return (uint32_t)max(s, 0);
}
// 2^(127 - s): exact for every byte scale_byte gives (0 .. 247).
__device__ __forceinline__ float scale_inverse(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// Two values as e4m3 (lo in the low byte); what is not finite becomes NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  const float nan = __uint_as_float(0x7FFFFFFFu);
  lo = fabsf(lo) <= FLT_MAX ? lo : nan;
  hi = fabsf(hi) <= FLT_MAX ? hi : nan;
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
// int8 at a position: round to nearest even, saturating; NaN gives 0.
__device__ __forceinline__ uint32_t s8x4(float a, float b, float c, float d) {
  const float v[4] = {a, b, c, d};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int r;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(v[i]));
    w |= ((uint32_t)r & 0xFFu) << (8 * i);
  }
  return w;
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ---------------------------------------------------------------- quantise
// Rows in blocks of 1 x 128: 16 lanes per block, eight values per lane. Bound by HBM.
constexpr int kQThreads = 256;
constexpr int kQUnroll = 4;  // blocks per half-warp, so four 16-byte loads per lane are in flight
template <typename T>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T* __restrict__ x, long long ldx, int K, int kb, long long blocks, uint8_t* __restrict__ q,
                         long long ldq, uint8_t* __restrict__ scale, long long lds) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, l16 = lane & 15;
  const long long hw = ((long long)blockIdx.x * kQThreads + threadIdx.x) >> 4;  // half-warp
  const long long hws = (long long)gridDim.x * (kQThreads / 16);
  for (long long b0 = hw; (b0 & ~1LL) < blocks; b0 += hws * kQUnroll) {  // a warp's two halves leave together
    Vec8<T> v[kQUnroll];
    long long row[kQUnroll];
    int col[kQUnroll];
    bool ok[kQUnroll];
#pragma unroll
    for (int i = 0; i < kQUnroll; ++i) {
      const long long b = b0 + i * hws;
      row[i] = b / kb;
      col[i] = (int)(b - row[i] * kb) * kQBlock + l16 * 8;
      ok[i] = b < blocks && col[i] < K;
      if (ok[i]) v[i] = load8(x + row[i] * ldx + col[i]);
    }
#pragma unroll
    for (int i = 0; i < kQUnroll; ++i) {
      float f[8], top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = ok[i] ? to_f32(v[i].v[j]) : 0.f;
        top = fmaxf(top, finite_abs(f[j]));
      }
      const uint32_t s = scale_byte(half_warp_max(top));
      const float m = scale_inverse(s);
      if (ok[i]) {
        *reinterpret_cast<uint2*>(q + row[i] * ldq + col[i]) =
            make_uint2(e4m3x4(f[0] * m, f[1] * m, f[2] * m, f[3] * m), e4m3x4(f[4] * m, f[5] * m, f[6] * m, f[7] * m));
        if (l16 == 0) scale[row[i] * lds + col[i] / kQBlock] = (uint8_t)s;
      }
    }
  }
}

// A weight's 128 x 128 blocks: a CTA per block, eight 16-byte vectors per thread held in registers
// between the maximum and the rounding, so the weight is read once.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_tiles_kernel(const T* __restrict__ x, long long ldx, int M, int K, uint8_t* __restrict__ q, long long ldq,
                          uint8_t* __restrict__ scale, long long lds) {
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float tops[8];
  const int tid = threadIdx.x;
  const int col = blockIdx.x * kQBlock + (tid & 15) * 8;
  const long long row0 = (long long)blockIdx.y * kQBlock + (tid >> 4);
  Vec8<T> v[8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col < K && row0 + 16 * i < M) v[i] = load8(x + (row0 + 16 * i) * ldx + col);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col < K && row0 + 16 * i < M) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_abs(to_f32(v[i].v[j])));
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, tops[i]);
  const uint32_t s = scale_byte(top);
  const float m = scale_inverse(s);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col < K && row0 + 16 * i < M) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = to_f32(v[i].v[j]) * m;
      *reinterpret_cast<uint2*>(q + (row0 + 16 * i) * ldq + col) =
          make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
    }
  if (tid == 0) scale[(long long)blockIdx.y * lds + blockIdx.x] = (uint8_t)s;
}

// ---------------------------------------------------------------- norm
struct NormParams {
  const void* x;         // [M][K]
  const void* residual;  // [M][K] or null
  const void* weight;    // [K]
  void* h;               // [M][K]: x + residual rounded to the inputs' type; null without a residual
  uint8_t* q;            // e4m3 or int8 [M][K]
  uint8_t* scale;        // [M][ceil(K/128)]; null: int8 at `position`
  long long ldx, ldr, ldh, ldq, lds;
  int M, K;
  float eps, unit;       // unit: 2^position
};

// A CTA per row (the grid strides over the rows): V vectors of eight values per thread stay in
// registers between the sum of squares and the output, so the row is read once. Bound by HBM for
// many rows, by the latency of one load, two barriers and one store for few.
template <typename T, typename W, int V>
__global__ void __launch_bounds__(V <= 2 ? 1024 : 512) norm_quant_kernel(const __grid_constant__ NormParams p) {
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float part[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const T* xs = static_cast<const T*>(p.x);
  const T* rs = static_cast<const T*>(p.residual);
  const W* ws = static_cast<const W*>(p.weight);
  T* hs = static_cast<T*>(p.h);
  int buf = 0;
  for (long long row = blockIdx.x; row < p.M; row += gridDim.x, buf ^= 1) {
    float f[V][8];
    float sum = 0.f;
    Vec8<T> a[V], r[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      if (col < p.K) {
        a[i] = load8(xs + row * p.ldx + col);
        if (rs) r[i] = load8(rs + row * p.ldr + col);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      const bool ok = col < p.K;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[i][j] = ok ? to_f32(a[i].v[j]) : 0.f;
        if (rs && ok) f[i][j] += to_f32(r[i].v[j]);
        sum = fmaf(f[i][j], f[i][j], sum);
      }
      if (rs && ok) {
        Vec8<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = from_f32<T>(f[i][j]);
        store8(hs + row * p.ldh + col, o);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) part[buf][warp] = sum;
    __syncthreads();  // the other buffer is free: every thread has passed this row's barrier only after reading it
    sum = lane < warps ? part[buf][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float rstd = 1.f / sqrtf(sum / (float)p.K + p.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      const bool ok = col < p.K;
      float top = 0.f;
      if (ok) {
        const Vec8<W> w = load8(ws + col);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          f[i][j] = f[i][j] * rstd * to_f32(w.v[j]);
          top = fmaxf(top, finite_abs(f[i][j]));
        }
      }
      uint2 o;
      if (p.scale) {
        const uint32_t s = scale_byte(half_warp_max(top));
        const float m = scale_inverse(s);
        o = make_uint2(e4m3x4(f[i][0] * m, f[i][1] * m, f[i][2] * m, f[i][3] * m),
                       e4m3x4(f[i][4] * m, f[i][5] * m, f[i][6] * m, f[i][7] * m));
        if (ok && (lane & 15) == 0) p.scale[row * p.lds + col / kQBlock] = (uint8_t)s;
      } else {
        const float m = p.unit;
        o = make_uint2(s8x4(f[i][0] * m, f[i][1] * m, f[i][2] * m, f[i][3] * m),
                       s8x4(f[i][4] * m, f[i][5] * m, f[i][6] * m, f[i][7] * m));
      }
      if (ok) *reinterpret_cast<uint2*>(p.q + row * p.ldq + col) = o;
    }
  }
}

// ---------------------------------------------------------------- products
// tcgen05.mma kind::mxf8f6f4 with block scales. The weight rows are the MMA's M (128 rows: one
// scale for the whole block), the tokens its N, so a single token costs a 16-column MMA and a
// long prompt a 240-column one in the same kernel. Each MMA takes 32 of K; the four of a
// 128-block use the same scale byte. A tile is MT blocks of 128 weight rows (swiglu: one block
// of gate rows and the up rows of the same outputs) by bn tokens.
//
// Scales reach the tensor core through TMEM: for 128 rows, four consecutive K-blocks' bytes of a
// row are one 32-bit word, lane r % 32, column r / 32, repeated in the four lane quarters. One
// warp gathers them from global memory into a 512-byte shared-memory image per 128 rows, and
// tcgen05.cp (32x128b, warpx4) brings that into TMEM, in order before the MMAs that read it.
//
// Few tokens leave few tiles: a cluster of `split` CTAs then shares a tile along K and adds its
// 32-bit parts in rank order over distributed shared memory.
constexpr int kFp8Epi = 8;                               // epilogue warps, two groups of four
constexpr int kFp8Threads = 32 * (kFp8Epi + 3);          // + TMA producer, MMA issuer, scale gatherer
constexpr int kFp8MaxStages = 12;
constexpr int kSfSlots = 4;                              // scale images in shared memory, 4 K-blocks each
constexpr int kSfSpan = 4;                               // K-blocks per scale image: one 32-bit word per row
constexpr int kSfAtom = 512;                             // bytes of one 128-row image
constexpr int kFp8Chunk = 16;                            // columns the epilogue stages at a time
constexpr int kFp8BarBytes = 512;
enum : int { FP8_LINEAR = 0, FP8_SWIGLU = 1 };

struct Fp8Params {
  alignas(64) CUtensorMap tx;     // x [M][K], box {128 B, bn rows}, SWIZZLE_128B
  alignas(64) CUtensorMap tw[2];  // w [N][K] (swiglu: gate, up), box {128 B, 128 rows}, SWIZZLE_128B
  int M, N, K;
  int bn, n_tiles, m_tiles, kblocks, split, kb_split;
  int stages, stage_bytes, sf_off, stg_off, bar_off;
  int acc_cols, nacc, tmem_cols;
  uint32_t idesc;
  const uint8_t* xs;
  const uint8_t* ws[2];
  long long ldxs, ldws[2];
  const uint8_t* w[2];  // the weights, for the L2 prefetch of few tokens; null: none
  long long ldw[2];
  int out_type;
  void* out;            // linear
  long long ldo;
  uint8_t* q;           // swiglu
  uint8_t* qs;
  long long ldq, ldqs;
};

// Instruction descriptor of tcgen05.mma kind::mxf8f6f4: e4m3 x e4m3 -> f32, both K-major, e8m0 scales.
__host__ __device__ constexpr uint32_t umma_idesc_mxf8(int m, int n) {
  return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= (A * scales) (B * scales)^T; `id` (0..3): the byte of the scale words that applies.
__device__ __forceinline__ void umma_mxf8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t id,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc | (id << 29) | (id << 4)), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// A 512-byte scale image (32 rows of 16 bytes) into four TMEM columns of every lane quarter.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(umma_desc(saddr, 128, 128)) : "memory");
}
// Four consecutive K-blocks' scale bytes of one row as a word, first block in the low byte; blocks
// at or past `end` read as 0 and are not touched.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* p, int kb, int end) {
  if (kb + 4 <= end && (reinterpret_cast<uintptr_t>(p + kb) & 3) == 0) return __ldg(reinterpret_cast<const uint32_t*>(p + kb));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (kb + i < end) w |= (uint32_t)__ldg(p + kb + i) << (8 * i);
  return w;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// One token's 128 outputs of a tile, four consecutive ones per lane.
template <typename T>
__device__ __forceinline__ void store_out4(T* o, int n, int N, float4 v) {
  const float f[4] = {v.x, v.y, v.z, v.w};
  if (n + 4 <= N && (reinterpret_cast<uintptr_t>(o + n) & (4 * sizeof(T) - 1)) == 0) {
    alignas(16) T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = from_f32<T>(f[i]);
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(o + n) = *reinterpret_cast<const uint2*>(t);
    else *reinterpret_cast<uint4*>(o + n) = *reinterpret_cast<const uint4*>(t);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < N) o[n + i] = from_f32<T>(f[i]);
  }
}
__device__ __forceinline__ void finish_linear(const Fp8Params& p, int m, int n, float4 v) {
  if (p.out_type == FT_BF16) store_out4(static_cast<__nv_bfloat16*>(p.out) + m * p.ldo, n, p.N, v);
  else if (p.out_type == FT_F16) store_out4(static_cast<__half*>(p.out) + m * p.ldo, n, p.N, v);
  else store_out4(static_cast<float*>(p.out) + m * p.ldo, n, p.N, v);
}
// silu(g) * u. The quotient's and the exponential's few units in the last place are far inside e4m3's 2^-4.
__device__ __forceinline__ float swiglu_value(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }
__device__ __forceinline__ void finish_swiglu(const Fp8Params& p, int m, int n, float4 g, float4 u) {
  float y[4] = {swiglu_value(g.x, u.x), swiglu_value(g.y, u.y), swiglu_value(g.z, u.z), swiglu_value(g.w, u.w)};
  const bool ok = n < p.N;  // N is a multiple of 16, n of 4
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, ok ? finite_abs(y[i]) : 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t s = scale_byte(top);
  const float r = scale_inverse(s);
  if (ok) {
    *reinterpret_cast<uint32_t*>(p.q + m * p.ldq + n) = e4m3x4(y[0] * r, y[1] * r, y[2] * r, y[3] * r);
    if ((n & 127) == 0) p.qs[m * p.ldqs + n / kQBlock] = (uint8_t)s;
  }
}

// MODE: FP8_LINEAR or FP8_SWIGLU; MT: blocks of 128 weight rows per tile (swiglu: 2, gate and up).
template <int MODE, int MT>
__global__ void __launch_bounds__(kFp8Threads, 1) fp8_gemm_kernel(const __grid_constant__ Fp8Params p) {
  constexpr int PW = kFp8Epi, MW = kFp8Epi + 1, SW = kFp8Epi + 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.bar_off);
  uint64_t* empty = full + kFp8MaxStages;
  uint64_t* sf_full = empty + kFp8MaxStages;
  uint64_t* sf_empty = sf_full + kSfSlots;
  uint64_t* acc_full = sf_empty + kSfSlots;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* done = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int rank = p.split > 1 ? (int)cluster_rank() : 0;
  const int tiles = p.n_tiles * p.m_tiles;
  const int tile0 = blockIdx.x / p.split, tstep = gridDim.x / p.split;
  const int kb0 = rank * p.kb_split, kb1 = min(p.kblocks, kb0 + p.kb_split);  // host: kb0 < kblocks for every rank
  const int sfb_groups = (p.bn + 127) / 128;
  const int sf_bytes = (MT + sfb_groups) * kSfAtom;

  grid_dep_launch();
  if (p.w[0] && tid < 128) {
    // few tokens: this CTA's weights, asked into L2 while the previous kernel drains (a hint; no value is used)
#pragma unroll
    for (int b = 0; b < MT; ++b) {
      const int src = MODE == FP8_SWIGLU ? b : 0;
      const long long row = (long long)(tile0 % p.n_tiles) * (MODE == FP8_SWIGLU ? 128 : 128 * MT) +
                            (MODE == FP8_SWIGLU ? 0 : b * 128) + tid;
      const int k0 = kb0 * 128, k1 = min(p.K, kb1 * 128);
      if (row < p.N) bulk_prefetch_l2(p.w[src] + row * p.ldw[src] + k0, (uint32_t)(k1 - k0));
    }
  }
  if (warp == MW) {
    tmem_alloc(tmem_slot, p.tmem_cols);
    tmem_relinquish();
  }
  if (tid == PW * 32) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(&sf_full[s], 1);
      mbar_init(&sf_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kFp8Epi);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tx) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tw[0]) : "memory");
    if (MODE == FP8_SWIGLU) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tw[1]) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();  // x, the scales, and whatever still reads the outputs, from here on

  if (warp == PW) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = tile0; ok && t < tiles; t += tstep) {
        const int mt = t / p.n_tiles, nt = t - mt * p.n_tiles;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * p.stage_bytes;
          mbar_arrive_expect_tx(&full[s], (uint32_t)p.stage_bytes);
#pragma unroll
          for (int b = 0; b < MT; ++b) {
            if (MODE == FP8_SWIGLU) tma_load_2d(st + b * kGemmABlock, &p.tw[b], kb * 128, nt * 128, &full[s]);
            else tma_load_2d(st + b * kGemmABlock, &p.tw[0], kb * 128, (nt * MT + b) * 128, &full[s]);
          }
          tma_load_2d(st + MT * kGemmABlock, &p.tx, kb * 128, mt * p.bn, &full[s]);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == SW) {
    // ------------------------------------------------------------ scale gatherer
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = tile0; ok && t < tiles; t += tstep) {
      const int mt = t / p.n_tiles, nt = t - mt * p.n_tiles;
      const uint8_t* wrow[MT];
      const uint8_t* xrow[2][4];
#pragma unroll
      for (int b = 0; b < MT; ++b) {
        const int src = MODE == FP8_SWIGLU ? b : 0;
        const long long r = MODE == FP8_SWIGLU ? nt : (long long)nt * MT + b;
        wrow[b] = r * 128 < p.N ? p.ws[src] + r * p.ldws[src] : nullptr;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = g * 128 + j * 32 + lane;
          const long long m = (long long)mt * p.bn + r;
          xrow[g][j] = r < p.bn && m < p.M ? p.xs + m * p.ldxs : nullptr;
        }
      for (int kb = kb0; kb < kb1; kb += kSfSpan) {
        uint32_t w[MT], x[2][4];
#pragma unroll
        for (int b = 0; b < MT; ++b) w[b] = wrow[b] ? scale_word(wrow[b], kb, p.kblocks) : 0;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[g][j] = xrow[g][j] ? scale_word(xrow[g][j], kb, p.kblocks) : 0;
        if (!mbar_wait(&sf_empty[s], ph ^ 1)) {
          ok = false;
          break;
        }
        uint8_t* im = smem + p.sf_off + s * sf_bytes;
#pragma unroll
        for (int b = 0; b < MT; ++b)
          *reinterpret_cast<uint4*>(im + b * kSfAtom + lane * 16) = make_uint4(w[b], w[b], w[b], w[b]);
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (g < sfb_groups)
            *reinterpret_cast<uint4*>(im + (MT + g) * kSfAtom + lane * 16) = make_uint4(x[g][0], x[g][1], x[g][2], x[g][3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sf_full[s]);
        if (++s == kSfSlots) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == MW) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int s = 0, acc = 0, ss = 0;
      uint32_t ph = 0, aph = 0, sph = 0, sfbuf = 0;
      bool ok = true, issued = false;
      const uint32_t sf_cols = 4 * (MT + sfb_groups);
      for (int t = tile0; ok && t < tiles; t += tstep) {
        if (!mbar_wait(&acc_empty[acc], aph ^ 1)) break;
        tc_fence_after();
        const uint32_t d0 = tmem + acc * p.acc_cols;
        uint32_t sf = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          const int id = (kb - kb0) % kSfSpan;
          if (id == 0) {
            if (!mbar_wait(&sf_full[ss], sph)) {
              ok = false;
              break;
            }
            tc_fence_after();
            sf = tmem + p.nacc * p.acc_cols + sfbuf * sf_cols;  // two sets of columns in turn
            const uint32_t im = smem_u32(smem + p.sf_off + ss * sf_bytes);
            for (int g = 0; g < MT + sfb_groups; ++g) tmem_cp_scales(sf + 4 * g, im + g * kSfAtom);
            sfbuf ^= 1;
          }
          if (!mbar_wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + s * p.stage_bytes);
          const int ksteps = min(4, (p.K - kb * 128 + 31) / 32);
          for (int j = 0; j < ksteps; ++j) {
            const uint64_t bd = umma_desc_sw128(st + MT * kGemmABlock + j * 32);
#pragma unroll
            for (int b = 0; b < MT; ++b)
              umma_mxf8(d0 + b * p.bn, umma_desc_sw128(st + b * kGemmABlock + j * 32), bd, p.idesc, id, sf + 4 * b,
                        sf + 4 * MT, (kb > kb0 || j) ? 1u : 0u);
          }
          issued = true;
          umma_commit(&empty[s]);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
          if (id == kSfSpan - 1 || kb == kb1 - 1) {
            umma_commit(&sf_empty[ss]);
            if (++ss == kSfSlots) {
              ss = 0;
              sph ^= 1;
            }
          }
        }
        if (!ok) break;
        umma_commit(&acc_full[acc]);
        if (++acc == p.nacc) {
          acc = 0;
          aph ^= 1;
        }
      }
      if (issued) {
        umma_commit(done);  // every MMA this CTA issued has finished before TMEM is released
        mbar_wait(done, 0);
      }
    }
  } else if (p.split == 1) {
    // ------------------------------------------------------------ epilogue
    // A group of four warps (one per TMEM lane quarter) moves kFp8Chunk columns through shared
    // memory, so that a warp then holds one token's 128 outputs and stores them as one run.
    // After a wait that gave up every warp runs on without work: all reach every barrier.
    constexpr int NB = MODE == FP8_SWIGLU ? 2 : 1;  // blocks staged together
    const int q = warp & 3, g = warp >> 2;
    float* stg = reinterpret_cast<float*>(smem + p.stg_off) + g * (NB * kFp8Chunk * 128);
    const int nch = p.bn / kFp8Chunk;
    const int items = MODE == FP8_SWIGLU ? nch : MT * nch;
    int acc = 0;
    uint32_t aph = 0;
    bool ok = true;
    for (int t = tile0; t < tiles; t += tstep) {
      ok = mbar_wait(&acc_full[acc], aph) && ok;
      tc_fence_after();
      const int mt = t / p.n_tiles, nt = t - mt * p.n_tiles;
      const uint32_t base = tmem + acc * p.acc_cols + ((uint32_t)(q * 32) << 16);
      for (int i = g; i < items; i += kFp8Epi / 4) {
        const int blk = MODE == FP8_SWIGLU ? 0 : i / nch, c = i - blk * nch;
        uint32_t v[NB][16];
#pragma unroll
        for (int b = 0; b < NB; ++b) tmem_ld16(base + (blk + b) * p.bn + c * kFp8Chunk, v[b]);
        tmem_ld_wait();
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < kFp8Chunk; ++e) stg[(b * kFp8Chunk + e) * 128 + q * 32 + lane] = __uint_as_float(v[b][e]);
        group_sync(1 + g);
#pragma unroll
        for (int e = q; e < kFp8Chunk; e += 4) {
          const int m = mt * p.bn + c * kFp8Chunk + e;
          if (!ok || m >= p.M) continue;  // warp-uniform
          const float4 a = *reinterpret_cast<const float4*>(stg + e * 128 + lane * 4);
          if (MODE == FP8_SWIGLU)
            finish_swiglu(p, m, nt * 128 + lane * 4, a, *reinterpret_cast<const float4*>(stg + (kFp8Chunk + e) * 128 + lane * 4));
          else
            finish_linear(p, m, (nt * MT + blk) * 128 + lane * 4, a);
        }
        group_sync(1 + g);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (++acc == p.nacc) {
        acc = 0;
        aph ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------ this rank's part of a split tile
    const int q = warp & 3, g = warp >> 2;
    float* red = reinterpret_cast<float*>(smem);  // [MT * bn][128] over the stages, which every MMA has read
    if (mbar_wait(&acc_full[0], 0)) {
      tc_fence_after();
      const uint32_t base = tmem + ((uint32_t)(q * 32) << 16);
      for (int c = g; c < MT * p.bn / 16; c += kFp8Epi / 4) {
        uint32_t v[16];
        tmem_ld16(base + c * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) red[(c * 16 + e) * 128 + q * 32 + lane] = __uint_as_float(v[e]);
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (p.split > 1) {
    cluster_sync();
    if (warp < kFp8Epi && !wait_timed_out()) {
      const int mt = tile0 / p.n_tiles, nt = tile0 - mt * p.n_tiles;
      for (int c = rank * kFp8Epi + warp; c < p.bn; c += p.split * kFp8Epi) {
        const int m = mt * p.bn + c;
        if (m >= p.M) break;
        float4 v[MT];
#pragma unroll
        for (int b = 0; b < MT; ++b) {
          v[b] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int r = 0; r < p.split; ++r) {
            const float4 a = ld_cluster_f4(cluster_addr(smem + ((b * p.bn + c) * 128 + lane * 4) * 4, r));
            v[b].x += a.x;
            v[b].y += a.y;
            v[b].z += a.z;
            v[b].w += a.w;
          }
        }
        if constexpr (MODE == FP8_SWIGLU) finish_swiglu(p, m, nt * 128 + lane * 4, v[0], v[MT - 1]);
        else
#pragma unroll
          for (int b = 0; b < MT; ++b) finish_linear(p, m, (nt * MT + b) * 128 + lane * 4, v[b]);
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its shared memory
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MW) tmem_dealloc(tmem, p.tmem_cols);
}

}  // namespace ixb
