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
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// Eight consecutive values as they lie in memory, 16-byte aligned, two (fp32: one) per word.
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
__device__ __forceinline__ void unpack8(const Vec8<__nv_bfloat16>& v, float (&f)[8]) {
  const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of the fp32
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void unpack8(const Vec8<__half>& v, float (&f)[8]) {
  const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void unpack8(const Vec8<float>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(v.w[i].x);
    f[4 * i + 1] = __uint_as_float(v.w[i].y);
    f[4 * i + 2] = __uint_as_float(v.w[i].z);
    f[4 * i + 3] = __uint_as_float(v.w[i].w);
  }
}
__device__ __forceinline__ void pack8(const float (&f)[8], Vec8<__nv_bfloat16>& v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<__nv_bfloat162*>(&w[i]) = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  v.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack8(const float (&f)[8], Vec8<__half>& v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<__half2*>(&w[i]) = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  v.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack8(const float (&f)[8], Vec8<float>& v) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v.w[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                        __float_as_uint(f[4 * i + 3]));
}

// Two fp32 operations in one instruction (sm_100a), over eight values.
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split_pair(unsigned long long v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ void add8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(a[i], a[i + 1])), "l"(pair_of(b[i], b[i + 1])));
    split_pair(r, a[i], a[i + 1]);
  }
}
__device__ __forceinline__ void mul8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(a[i], a[i + 1])), "l"(pair_of(b[i], b[i + 1])));
    split_pair(r, a[i], a[i + 1]);
  }
}
__device__ __forceinline__ void mul8(float (&a)[8], float b) {
  const float s[8] = {b, b, b, b, b, b, b, b};
  mul8(a, s);
}
__device__ __forceinline__ unsigned long long squares8(const float (&a)[8], unsigned long long sum) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const unsigned long long v = pair_of(a[i], a[i + 1]);
    asm("fma.rn.f32x2 %0, %1, %1, %0;" : "+l"(sum) : "l"(v));
  }
  return sum;
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
// Two values as e4m3 (lo in the low byte): nearest even, past 448 to 448, NaN to NaN. Infinities have to
// be NaN already (no_infinity).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
__device__ __forceinline__ float no_infinity(float v) { return fabsf(v) <= FLT_MAX ? v : __uint_as_float(0x7FFFFFFFu); }
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

// The largest finite |v| of the block of 128 values that a half-warp holds, eight per lane. fmaxf passes over
// NaN; an infinity, rare, sends the warp through the finite values once more and turns it into NaN.
__device__ __forceinline__ float block_top(float (&f)[8]) {
  float top = fabsf(f[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) top = fmaxf(top, fabsf(f[j]));
  top = half_warp_max(top);
  if (__any_sync(0xffffffffu, !(top <= FLT_MAX))) {
    top = finite_abs(f[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, finite_abs(f[j]));
    top = half_warp_max(top);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = no_infinity(f[j]);
  }
  return top;
}
__device__ __forceinline__ uint2 round8(float (&f)[8], float m) {
  mul8(f, m);
  return make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
}

// ---------------------------------------------------------------- quantise
// The pointers carry no __restrict__: the kernel before may still be writing x when one of these starts, so its
// loads must not become loads of read-only data.
// Rows in blocks of 1 x 128: 16 lanes per block, eight values per lane. Bound by HBM (11008 x 4096: 25.3 us in
// bf16, 5.3 TB/s, 35.5 in fp32, 6.4).
constexpr int kQThreads = 256;
constexpr int kQUnroll = 4;  // blocks per half-warp, so four 16-byte loads per lane are in flight
template <typename T>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T* x, long long ldx, int K, FastDiv kb, uint32_t blocks, uint8_t* q, long long ldq, uint8_t* scale,
                         long long lds) {
  grid_dep_launch();
  grid_dep_wait();
  const int l16 = threadIdx.x & 15;
  const uint32_t hws = gridDim.x * (kQThreads / 16);  // half-warps; even, so a warp's two halves leave together
  for (uint32_t b0 = (blockIdx.x * kQThreads + threadIdx.x) >> 4; (b0 & ~1u) < blocks; b0 += hws * kQUnroll) {
    Vec8<T> v[kQUnroll];
    uint32_t row[kQUnroll];
    int col[kQUnroll];
    bool ok[kQUnroll];
#pragma unroll
    for (int i = 0; i < kQUnroll; ++i) {
      const uint32_t b = b0 + i * hws;  // below 2^31 + 4 * 2^22: no wrap
      row[i] = fdiv(b, kb);
      col[i] = (int)(b - row[i] * kb.d) * kQBlock + l16 * 8;
      ok[i] = b < blocks && col[i] < K;
      v[i] = ok[i] ? load8(x + row[i] * ldx + col[i]) : Vec8<T>{};
    }
#pragma unroll
    for (int i = 0; i < kQUnroll; ++i) {
      float f[8];
      unpack8(v[i], f);
      const uint32_t s = scale_byte(block_top(f));
      if (ok[i]) {
        *reinterpret_cast<uint2*>(q + row[i] * ldq + col[i]) = round8(f, scale_inverse(s));
        if (l16 == 0) scale[row[i] * lds + col[i] / kQBlock] = (uint8_t)s;
      }
    }
  }
}

// A weight's 128 x 128 blocks: a CTA per block, V vectors of eight per thread held in registers, as they lie
// in memory, between the maximum and the rounding, so the weight is read once. Bound by HBM: four
// CTAs' loads are in flight on an SM. (Kept unpacked, the values spill or leave room for two CTAs:
// 38 and 31 us for 11008 x 4096 bf16 instead of 21.5, 6.3 TB/s; fp32, with two, 34.6 us, 6.5 TB/s.)
constexpr int kTileThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 2 ? 4 : 2)
    quantize_tiles_kernel(const T* x, long long ldx, int M, int K, uint8_t* q, long long ldq, uint8_t* scale, long long lds) {
  constexpr int V = 128 * 128 / 8 / kTileThreads, kStep = kTileThreads / 16;  // rows between a thread's vectors
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float tops[2][kTileThreads / 32];
  const int tid = threadIdx.x;
  const int col = blockIdx.x * kQBlock + (tid & 15) * 8;
  const long long row0 = (long long)blockIdx.y * kQBlock + (tid >> 4);
  auto in = [&](int i) { return col < K && row0 + kStep * i < M; };
  auto block_top = [&](float top, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((tid & 31) == 0) part[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTileThreads / 32; ++i) top = fmaxf(top, part[i]);
    return top;
  };
  Vec8<T> v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = in(i) ? load8(x + (row0 + kStep * i) * ldx + col) : Vec8<T>{};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float f[8];
    unpack8(v[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(f[j]));
  }
  top = block_top(top, tops[0]);
  const bool infinite = !(top <= FLT_MAX);  // the same in every thread
  if (infinite) {  // rare: the finite values alone, read again
    top = 0.f;
#pragma unroll 1
    for (int i = 0; i < V; ++i)
      if (in(i)) {
        float f[8];
        unpack8(load8(x + (row0 + kStep * i) * ldx + col), f);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_abs(f[j]));
      }
    top = block_top(top, tops[1]);
  }
  const uint32_t s = scale_byte(top);
  const float m = scale_inverse(s);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < (int)(sizeof(T) / 2); ++j)  // opaque, so that nothing unpacked is kept
      asm volatile("" : "+r"(v[i].w[j].x), "+r"(v[i].w[j].y), "+r"(v[i].w[j].z), "+r"(v[i].w[j].w));
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float f[8];
    unpack8(v[i], f);
    if (infinite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = no_infinity(f[j]);
    }
    if (in(i)) *reinterpret_cast<uint2*>(q + (row0 + kStep * i) * ldq + col) = round8(f, m);
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

// A CTA per row, the grid striding over the rows: V vectors of eight values per thread stay in registers
// between the sum of squares and the output, so the row is read once. With many rows HBM bounds it,
// and the next row's loads (without a residual the next two rows') are issued before this row's barrier, so
// that they are in flight while it is reduced and rounded, and the weight stays in registers (V up to
// 2 and 16-bit values: more would spill): 8192 x 4096 bf16 with a residual 38.5 us (6.1 TB/s), without one 28.0 us
// (3.6 TB/s, bound by instructions), fp32 70 us (6.2 TB/s). V 8, for rows above 16384 values, spills even so (80 to
// 352 bytes a thread): 512 x 32768 with a residual 33.4 us in bf16 (3.5 TB/s), 65.3 in fp32 (3.3). With few rows:
// one load, one barrier and one store.
template <typename T, typename W, int V>
__global__ void __launch_bounds__(V <= 2 ? 1024 : 512) norm_quant_kernel(const __grid_constant__ NormParams p) {
  constexpr bool kAhead = V <= 2 && sizeof(T) == 2;
  grid_dep_launch();
  grid_dep_wait();
  __shared__ float part[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  int wide = 1;  // warps, rounded up to a power of two; the parts past them stay 0
  while (wide < warps) wide *= 2;
  if (tid < 32) part[0][tid] = part[1][tid] = 0.f;
  __syncthreads();
  const float inv_k = 1.f / (float)p.K;
  const T* xs = static_cast<const T*>(p.x);
  const T* rs = static_cast<const T*>(p.residual);
  const W* ws = static_cast<const W*>(p.weight);
  T* hs = static_cast<T*>(p.h);
  // a: the row's x; b: its residual, or, without one, the x of the CTA's next row
  Vec8<T> a[V], b[V];
  auto load = [&](Vec8<T>(&v)[V], const T* base, long long ld, long long row) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      v[i] = col < p.K && row < p.M ? load8(base + row * ld + col) : Vec8<T>{};
    }
  };
  const long long step = gridDim.x;
  if (kAhead) {
    load(a, xs, p.ldx, blockIdx.x);
    load(b, rs ? rs : xs, rs ? p.ldr : p.ldx, rs ? blockIdx.x : blockIdx.x + step);
  }
  Vec8<W> wv[V];
  auto load_weight = [&] {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      wv[i] = col < p.K ? load8(ws + col) : Vec8<W>{};
    }
  };
  if (kAhead) load_weight();
  int buf = 0;
  for (long long row = blockIdx.x; row < p.M; row += step, buf ^= 1) {
    if (!kAhead) {
      load(a, xs, p.ldx, row);
      if (rs) load(b, rs, p.ldr, row);
    }
    float f[V][8];
    unsigned long long sum2 = 0;  // two partial sums
#pragma unroll
    for (int i = 0; i < V; ++i) {
      unpack8(a[i], f[i]);
      if (rs) {
        float t[8];
        unpack8(b[i], t);
        add8(f[i], t);
      }
      sum2 = squares8(f[i], sum2);
    }
    float sum, odd;
    split_pair(sum2, sum, odd);
    sum += odd;
    if (rs) {  // before the next row's loads: h may be x or the residual, whose rows a CTA reads alone
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int col = (i * blockDim.x + tid) * 8;
        if (col < p.K) {
          Vec8<T> o;
          pack8(f[i], o);
          store8(hs + row * p.ldh + col, o);
        }
      }
    }
    if (!kAhead) {
      load_weight();
    } else if (rs) {
      load(a, xs, p.ldx, row + step);
      load(b, rs, p.ldr, row + step);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = b[i];
      load(b, xs, p.ldx, row + 2 * step);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) part[buf][warp] = sum;
    // h * weight and the blocks' maxima do not need the row's sum: the root is one factor of a whole row,
    // and rounding keeps the order of products with it
    float top[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float w[8];
      unpack8(wv[i], w);
      mul8(f[i], w);  // past the row's end both are 0, and nothing is stored
      if (p.scale) top[i] = block_top(f[i]);
    }
    __syncthreads();  // the other buffer is free: every thread has passed this row's barrier only after reading it
    sum = part[buf][lane & (wide - 1)];
    for (int o = wide >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float mean = fmaf(sum, inv_k, p.eps);
    float rstd = rsqrtf(mean);
    if (mean <= FLT_MAX) rstd *= fmaf(-0.5f * mean * rstd, rstd, 1.5f);  // a Newton step: two units in the last place to one
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = (i * blockDim.x + tid) * 8;
      const bool ok = col < p.K;
      uint2 o;
      mul8(f[i], rstd);
      if (p.scale) {
        const uint32_t s = scale_byte(fmaxf(top[i] * rstd, 0.f));  // a NaN root: no finite value, scale byte 0
        o = round8(f[i], scale_inverse(s));
        if (ok && (lane & 15) == 0) p.scale[row * p.lds + col / kQBlock] = (uint8_t)s;
      } else {
        mul8(f[i], p.unit);
        o = make_uint2(s8x4(f[i][0], f[i][1], f[i][2], f[i][3]), s8x4(f[i][4], f[i][5], f[i][6], f[i][7]));
      }
      if (ok) *reinterpret_cast<uint2*>(p.q + row * p.ldq + col) = o;
    }
  }
}

// ---------------------------------------------------------------- products
// tcgen05.mma kind::mxf8f6f4 with block scales. The weight rows are the MMA's M (128 rows: one
// scale for the whole block), the tokens its N, so a single token costs a 16-column MMA and a
// long prompt a 224-column one in the same kernel. Each MMA takes 32 of K; the four of a
// 128-block use the same scale byte. A tile is MT blocks of 128 weight rows (swiglu: one block
// of gate rows and the up rows of the same outputs) by bn tokens.
//
// Scales reach the tensor core through TMEM: for 128 rows, four consecutive K-blocks' bytes of a
// row are one 32-bit word, lane r % 32, column r / 32, repeated in the four lane quarters. One
// warp gathers them from global memory into a 512-byte shared-memory image per 128 rows, and
// tcgen05.cp (32x128b, warpx4) brings that into TMEM, in order before the MMAs that read it.
//
// Two forms. Few tokens (CG 1): tiles of at most 128 tokens, one per CTA or cluster; a cluster of up to
// eight CTAs shares a tile along K and adds its 32-bit parts in rank order over distributed shared
// memory; shared memory and registers leave room for two CTAs per SM, so the next kernel's start
// overlaps this one's end. HBM bounds it (the weights are read once), with ~3 us of start and end:
// 1 x 4096 x 4096 5.7 us, 23 x 4096 x 11008 11.9 us (3.8 TB/s), 8 x 11008 x 4096 gate/up 18.5 us (4.9 TB/s).
// (Asking the weights into L2 before waiting for the previous kernel, as the W4A8 GEMV does, made the last of
// these 9 % slower and the others no faster.)
// Many tokens (CG 2): persistent pairs of CTAs, tiles of 256 weight rows x 224 tokens with two accumulators
// (or 512 rows and one, where that is one round). The tensor cores bound it, and in a long run the board's
// 1000 W: 8192 x 11008 x 4096 takes 262 us (2.8 PFLOP/s) in a burst and 318 us in a long run, at ~1.05 GHz, where
// the MMAs alone would take 300. A prompt chunk is bound by its operands' arrival and by what of the MMAs does
// not overlap it: 512 x 4096 x 11008 takes 0.229 us for a K-block of 128 tokens, 0.182 without the MMAs and 0.146
// without the loads.
// The tensor cores cut a running sum where an fp32 adder rounds, about once per K-block: 2e-8 to 3e-8 of the
// result's norm for each K-block of a chain. Taken as it is: with K = 65536 in one chain it is 1.7e-5, far below
// the rounding of a 16-bit or e4m3 output, and shorter chains would drain each accumulator several times per tile.
constexpr int kFp8Epi = 8;                               // epilogue warps, two groups of four
constexpr int kFp8Threads = 32 * (kFp8Epi + 3);          // + TMA producer, MMA issuer, scale gatherer
constexpr int kFp8MaxStages = 12;
constexpr int kFp8MaxSplit = 8;                          // CTAs that share a tile along K: a portable cluster
constexpr int kFp8FewTokens = 128;                       // tokens per tile of the split form
constexpr int kSfSlots = 2;                              // scale images in shared memory
constexpr int kSfSpan = 16;                              // K-blocks per image: four 32-bit words per row
constexpr int kSfAtom = 512;                             // bytes of four K-blocks' words of 128 rows
// swiglu pairs: each epilogue warp's two buffers of the peer's columns, and of the maxima; their barriers after
// the others
constexpr int kFp8Chunk = 16;
constexpr int kFp8WarpSwap = kFp8Chunk * 32 * 4;  // one warp's columns: 16 tokens x 32 outputs
constexpr int kFp8SwapBytes = kFp8Epi * 2 * kFp8WarpSwap;
constexpr int kFp8TopBytes = 2 * 2 * kFp8Chunk * 4 * 4;
constexpr int kFp8SwapBar = 384;
constexpr int kFp8BarBytes = 512;
// A TMEM allocation waits, without a limit, for the columns that other CTAs of the SM hold, and the CTAs of a
// cluster wait for one another. Two clusters on two streams must not each hold columns on one SM that the other
// needs on another: so a CTA of the few-token form takes at most half of TMEM, and at least the shared memory
// that lets two CTAs onto an SM and no third; a CTA of a pair takes all shared memory and is alone.
constexpr int kFp8FewTmem = 256;
constexpr int kSmShared = 228 * 1024;  // an SM's shared memory; the system takes 1 KB of it per CTA
constexpr int kFp8FewShared = kSmShared / 3 - 1024 + 128;
static_assert(3 * (kFp8FewShared + 1024) > kSmShared, "no third CTA");
enum : int { FP8_LINEAR = 0, FP8_SWIGLU = 1 };

struct Fp8Params {
  alignas(64) CUtensorMap tx;     // x [M][K], box {128 B, bn rows}, SWIZZLE_128B
  alignas(64) CUtensorMap tw[2];  // w [N][K] (swiglu: gate, up), box {128 B, 128 rows}, SWIZZLE_128B
  int M, N, K;
  int bn, n_tiles, n_group, m_tiles, kblocks, split, kb_split;
  int stages, stage_bytes, sf_off, stg_off, bar_off;
  int acc_cols, nacc, tmem_cols;
  uint32_t idesc;
  const uint8_t* xs;
  const uint8_t* ws[2];
  long long ldxs, ldws[2];
  int sf_words;  // every scale word is 4-byte aligned
  int out_type;
  void* out;            // linear
  long long ldo;
  uint8_t* q;           // swiglu
  uint8_t* qs;
  long long ldq, ldqs;
};

// K-blocks per stage. A turn of the MMA warp's loop (look at a barrier, elect, four MMAs, commit) takes ~440
// cycles, the MMAs of a pair's K-block with 128 tokens 256: two K-blocks to a turn where the pair's
// stages leave room (512 x 4096 x 11008 26.8 -> 24.5 us). The swiglu pairs hold their exchange too, and
// three stages of two measured slower than six of one (2048 x 11008 x 4096 146 us instead of 142).
__host__ __device__ constexpr int fp8_stage_blocks(int mode, int mt, int cg) {
  return cg == 2 && mt == 1 && mode == FP8_LINEAR ? 2 : 1;
}
// Instruction descriptor of tcgen05.mma kind::mxf8f6f4: e4m3 x e4m3 -> f32, both K-major, e8m0 scales.
__host__ __device__ constexpr uint32_t umma_idesc_mxf8(int m, int n) {
  return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= (A * scales) (B * scales)^T. Bits 29-30 and 4-5 of idesc choose the byte of A's and B's
// scale words that applies.
template <int CG>
__device__ __forceinline__ void umma_mxf8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// A 512-byte scale image (32 rows of 16 bytes) into four TMEM columns of every lane quarter; a pair's
// form takes each CTA's image into that CTA's TMEM.
template <int CG>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(umma_desc(saddr, 128, 128)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(umma_desc(saddr, 128, 128)) : "memory");
}

// Two-CTA pairs (cta_group::2). Every tcgen05 instruction of a kernel names the same group size.
template <int CG>
__device__ __forceinline__ void tmem_alloc_cg(uint32_t* slot, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(slot, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_cg(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(taddr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// Arrive on bar, in both CTAs of a pair at the same offset, once this thread's earlier tcgen05 work is done.
template <int CG>
__device__ __forceinline__ void umma_commit_cg(uint64_t* bar) {
  if constexpr (CG == 1) umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
// A tile of this CTA's operands into its own shared memory, its bytes counted on the barrier at `bar` (an
// address of the cluster's shared memory: the pair's leader).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(tm), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// A bounded wait without a suspend hint: every K-block hands a stage from the TMA to the tensor core and back,
// and waking from a long sleep is on that way. Same limit and flag as mbar_wait.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  if constexpr (CLUSTER)  // acquires what the cluster's other CTA released
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // does not wait
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_poll(uint64_t* bar, uint32_t parity) {
  if (mbar_try<CLUSTER>(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try<CLUSTER>(bar, parity)) return true;
    if ((i & 255) == 0 && (global_ns() - t0 > kWaitLimitNs || wait_timed_out())) break;
  }
  set_dev_error(DEV_ERR_WAIT_TIMEOUT);
  return false;
}
// A wait for what is on its way whether or not some other wait has given up (copies into this CTA's shared memory,
// MMAs into its TMEM): with the same limit, but the flag does not end it.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_settle(uint64_t* bar, uint32_t parity, unsigned long long t0 = 0) {  // t0: 0 is now
  if (mbar_try<CLUSTER>(bar, parity)) return true;
  if (t0 == 0) t0 = global_ns();
  while (!mbar_try<CLUSTER>(bar, parity))
    if (global_ns() - t0 > kWaitLimitNs) {
      set_dev_error(DEV_ERR_WAIT_TIMEOUT);
      return false;
    }
  return true;
}
// The wait's outcome as one value of the warp: a branch on it leaves the code after it uniform.
__device__ __forceinline__ bool warp_all(bool ok) { return __all_sync(0xffffffffu, ok); }
// A bounded wait for arrivals of the other CTA of a pair too.
template <int CG>
__device__ __forceinline__ bool mbar_wait_cg(uint64_t* bar, uint32_t parity) {
  return mbar_poll<CG == 2>(bar, parity);
}
// Four words into another CTA's shared memory, counted as 16 bytes on a barrier there: the store itself
// signals, so no release waits for this thread's earlier global stores.
__device__ __forceinline__ void st_async4(uint32_t to, const uint32_t* v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(bar)
               : "memory");
}
// Arrive on a barrier of either CTA: at cluster scope, publishing this thread's writes to the other CTA, and at
// CTA scope, for what the tensor core reads or has given (TMEM): a release at cluster scope waits for
// every global store this thread has in flight.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The next `bytes` (0..4) K-blocks' scale bytes of one row, 4-byte aligned, to a word in shared memory, first
// block in the low byte, zeros behind.
__device__ __forceinline__ void scale_copy(void* dst, const uint8_t* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
// The five aligned words that hold the 16 bytes from `src`; what lies at or past `end` (the matrix's) reads as 0.
// Predicated, without branches, so that the loads of many rows overlap. Returns whether `end` cuts one of
// the words: its bytes are missing.
// Plain loads in program order: the kernel that writes x's scales may still be running when this one starts, so
// they are no read-only data, and none may move above the wait for it.
__device__ __forceinline__ bool scale_words5(const uint8_t* src, const uint8_t* end, uint32_t (&w)[5]) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(src) & ~uintptr_t(3), e = reinterpret_cast<uintptr_t>(end);
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const uint32_t in = a + 4 * i + 4 <= e;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %2, 0;\n\t"
        "mov.b32 %0, 0;\n\t"
        "@p ld.global.b32 %0, [%1];\n\t}"
        : "=r"(w[i])
        : "l"(a + 4 * i), "r"(in)
        : "memory");
  }
  const uintptr_t t = e & ~uintptr_t(3);
  return t != e && t >= a && t < a + 20;
}
__device__ __forceinline__ void scale_last_bytes(const uint8_t* src, const uint8_t* end, uint32_t (&w)[5]) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(src) & ~uintptr_t(3), e = reinterpret_cast<uintptr_t>(end);
#pragma unroll
  for (int i = 0; i < 5; ++i)
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (a + 4 * i + j < e && a + 4 * i + 4 > e) w[i] |= (uint32_t)*reinterpret_cast<const uint8_t*>(a + 4 * i + j) << (8 * j);
}
// Where row i of a lane goes in four K-blocks' images: weight blocks first, then x's groups of 128 rows.
__device__ __forceinline__ int scale_place(int mt, int i) {
  return i < mt ? i * kSfAtom : mt * kSfAtom + (i - mt) / 4 * kSfAtom + (i - mt) % 4 * 4;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

// Up to 32 tokens' output n: a warp stores 32 consecutive outputs of each token.
template <typename T>
__device__ __forceinline__ void store_columns(T* out, long long ldo, const uint32_t (&v)[32], int n, int m0, int cols) {
  T* o = out + m0 * ldo + n;
  if (cols >= 32) {
#pragma unroll
    for (int e = 0; e < 32; ++e, o += ldo) *o = from_f32<T>(__uint_as_float(v[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e, o += ldo)
      if (e < cols) *o = from_f32<T>(__uint_as_float(v[e]));
  }
}
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
// g / (1 + exp(-g)) * u within a few units in the last place, for a value next to a rounding or scale border
// should fall on the side that exact arithmetic puts it. expf is CUDA's; the reciprocal is the
// hardware's with one Newton step, where that is finite (past 2^100 the quotient is far below any
// other output's).
__device__ __forceinline__ float swiglu_value(float g, float u) {
  const float d = 1.f + expf(-g);
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(d));
  r = d < 0x1p100f ? fmaf(fmaf(-d, r, 1.f), r, r) : r;
  return g * r * u;
}
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
    *reinterpret_cast<uint32_t*>(p.q + m * p.ldq + n) =
        e4m3x4(no_infinity(y[0]) * r, no_infinity(y[1]) * r, no_infinity(y[2]) * r, no_infinity(y[3]) * r);
    if ((n & 127) == 0) p.qs[m * p.ldqs + n / kQBlock] = (uint8_t)s;
  }
}

// The largest value of a warp (sm_100a reduces fp32 in one instruction).
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Up to 16 tokens' output n of the gate and up products, over a group of four warps that hold a token's 128
// outputs: each warp's maxima go through shared memory ([16 tokens][4 warps], two buffers in turn, so
// one barrier per call), lane c turns token c's into the scale, and every lane rounds. `between` runs
// once the inputs have been used.
template <typename F>
__device__ __forceinline__ void swiglu_columns(const Fp8Params& p, uint32_t (&gate)[kFp8Chunk], const uint32_t (&up)[kFp8Chunk],
                                               int n, int m0, int cols, float* tops, int bar, int q, int lane, F&& between) {
  const bool in = n < p.N;
  float mine = 0.f;
#pragma unroll
  for (int e = 0; e < kFp8Chunk; ++e) {
    const float y = swiglu_value(__uint_as_float(gate[e]), __uint_as_float(up[e]));
    const float top = warp_max(in ? finite_abs(y) : 0.f);
    gate[e] = __float_as_uint(no_infinity(y));
    mine = lane == e ? top : mine;
  }
  if (lane < kFp8Chunk) tops[lane * 4 + q] = mine;
  between();
  group_sync(bar);
  const float4 t = *reinterpret_cast<const float4*>(tops + (lane & (kFp8Chunk - 1)) * 4);
  const uint32_t s = scale_byte(fmaxf(fmaxf(t.x, t.y), fmaxf(t.z, t.w)));
  if (q == 0 && lane < cols) p.qs[(m0 + lane) * p.ldqs + n / kQBlock] = (uint8_t)s;
  const float inv = scale_inverse(s);
  uint8_t* o = p.q + m0 * p.ldq + n;
#pragma unroll
  for (int e = 0; e < kFp8Chunk; e += 2) {
    const uint32_t w = e4m3x2(__uint_as_float(gate[e]) * __shfl_sync(0xffffffffu, inv, e),
                              __uint_as_float(gate[e + 1]) * __shfl_sync(0xffffffffu, inv, e + 1));
    if (in && e < cols) *o = (uint8_t)w;
    o += p.ldq;
    if (in && e + 1 < cols) *o = (uint8_t)(w >> 8);
    o += p.ldq;
  }
}

// Tiles go through n in groups of p.n_group and through all m within a group, n first: the tiles in work at
// one time then form a near-square, and what they read (a group's weights, a few rows of x) is read
// from L2 by as few as can be (8192 x 11008 x 4096 takes 3 % longer through all of n first).
__device__ __forceinline__ void tile_at(const Fp8Params& p, int t, int& mt, int& nt) {
  const int per = p.n_group * p.m_tiles, g = t / per, r = t - g * per;
  const int size = min(p.n_group, p.n_tiles - g * p.n_group);
  mt = r / size;
  nt = g * p.n_group + r - mt * size;
}
template <int MODE, int MT, int CG>
__device__ __forceinline__ int weight_block(int nt, int pair, int b) {  // 128-row block b of this CTA's part of tile nt
  return MODE == FP8_SWIGLU ? nt : (nt * CG + pair) * MT + b;
}
template <int MODE, int CG>
__device__ __forceinline__ int weight_source(int pair, int b) {  // which weight it is a block of: 0 (gate), 1 (up)
  return MODE == FP8_SWIGLU ? (CG == 2 ? pair : b) : 0;
}
// MODE: FP8_LINEAR or FP8_SWIGLU; MT: blocks of 128 weight rows per tile and CTA. CG 2: a pair of CTAs
// shares a tile's tokens: each holds its own rows' operand, accumulators and epilogue and half of the
// tokens' operand, and the leader (rank 0) issues the MMAs of both, so each SM fetches half the token
// bytes per product. Swiglu: with CG 1 a CTA has a block of gate rows and the up rows of the same
// outputs (MT 2); with CG 2 the leader has the gate rows and the other CTA the up rows, so that each has
// room for two accumulators and the epilogue runs beside the next tile's MMAs.
template <int MODE, int MT, int CG>
__global__ void __launch_bounds__(kFp8Threads, CG == 1 ? 2 : 1) fp8_gemm_kernel(const __grid_constant__ Fp8Params p) {
  constexpr int PW = kFp8Epi, MW = kFp8Epi + 1, SW = kFp8Epi + 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform to the compiler too
  const int S = p.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.bar_off);
  uint64_t* empty = full + kFp8MaxStages;
  uint64_t* sf_full = empty + kFp8MaxStages;
  uint64_t* sf_empty = sf_full + kSfSlots;
  uint64_t* acc_full = sf_empty + kSfSlots;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* done = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int rank = CG == 1 ? (int)cluster_rank() : 0;  // part of K
  const int pair = CG == 2 ? (int)cluster_rank() : 0;  // part of the tile
  const int tiles = p.n_tiles * p.m_tiles;
  const int share = CG == 2 ? 2 : p.split;
  const int tile0 = blockIdx.x / share, tstep = gridDim.x / share;
  const int kb0 = rank * p.kb_split, kb1 = min(p.kblocks, kb0 + p.kb_split);  // host: kb0 < kblocks for every rank
  constexpr int kXRows = CG == 1 ? 4 : 8;  // x rows per lane of a scale image: bn is at most 128, or 256
  const int sfb_groups = CG == 1 ? 1 : (p.bn + 127) / 128;
  const int sf_quad = (MT + sfb_groups) * kSfAtom;  // four K-blocks' images
  constexpr int KS = fp8_stage_blocks(MODE, MT, CG);
  const int block_bytes = p.stage_bytes / KS;

  if (warp == MW) tmem_alloc_cg<CG>(tmem_slot, p.tmem_cols);
  if (tid == PW * 32) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSfSlots; ++s) {
      mbar_init(&sf_full[s], CG);
      mbar_init(&sf_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * kFp8Epi);
    }
    mbar_init(done, 1);
    if (MODE == FP8_SWIGLU && CG == 2)
      for (int b = 0; b < 2 * kFp8Epi; ++b) mbar_init(reinterpret_cast<uint64_t*>(smem + p.bar_off + kFp8SwapBar) + b, 1);
    fence_mbar_init();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tx) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tw[0]) : "memory");
    if (MODE == FP8_SWIGLU) asm volatile("prefetch.tensormap [%0];" ::"l"(&p.tw[1]) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_launch();  // not before this CTA has its TMEM: the next kernel's CTAs would hold theirs until this grid ends
  bool part_ok = true;
  grid_dep_wait();  // x, the scales, and whatever still reads the outputs, from here on

  if (warp == PW) {
    // ------------------------------------------------------------ TMA producer
    // This warp's and the MMA warp's loops run in all lanes and one elected lane issues, so addresses and
    // descriptors stay in uniform registers (with the loops inside `if (lane == 0)` 8192 x 11008 x 4096
    // takes 17 % longer).
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = tile0; ok && t < tiles; t += tstep) {
      int mt, nt;
      tile_at(p, t, mt, nt);
      for (int kb = kb0; kb < kb1; kb += KS) {
        if (!warp_all(mbar_poll(&empty[s], ph ^ 1))) {
          ok = false;
          break;
        }
        uint8_t* st = smem + s * p.stage_bytes;
        const int n = min(KS, kb1 - kb);
        if (elect_one()) {
          if (pair == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(CG * n * block_bytes));
          const uint32_t lead = CG == 2 ? cluster_addr(&full[s], 0) : 0;
#pragma unroll
          for (int k = 0; k < KS; ++k, st += block_bytes) {
            if (k >= n) break;
#pragma unroll
            for (int b = 0; b < MT; ++b) {
              const CUtensorMap* tw = &p.tw[weight_source<MODE, CG>(pair, b)];
              const int row = weight_block<MODE, MT, CG>(nt, pair, b) * 128;
              if (CG == 2) tma_load_2d_pair(st + b * kGemmABlock, tw, (kb + k) * 128, row, lead);
              else tma_load_2d(st + b * kGemmABlock, tw, (kb + k) * 128, row, &full[s]);
            }
            if (CG == 2) tma_load_2d_pair(st + MT * kGemmABlock, &p.tx, (kb + k) * 128, mt * p.bn + pair * (p.bn / 2), lead);
            else tma_load_2d(st + MT * kGemmABlock, &p.tx, (kb + k) * 128, mt * p.bn, &full[s]);
          }
        }
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    // The releases of the last stages, which the pair's leader sends to both CTAs, have arrived before this CTA
    // leaves: a signal still on its way would reach the shared memory of whoever has it next. After a wait
    // that gave up nothing may read the last stages, and their copies have to land all the same (a pair's count on
    // the leader's barriers, and its other CTA stays until the leader is done).
    const unsigned long long t0 = global_ns();
    for (int i = 0; i < S; ++i) {
      ok = ok && warp_all(mbar_poll(&empty[s], ph ^ 1));
      if (!ok && pair == 0) mbar_settle(&full[s], ph ^ 1, t0);
      if (++s == S) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == SW) {
    // ------------------------------------------------------------ scale gatherer
    // Words go straight from global to shared memory (cp.async, 4 bytes each, short or absent ones
    // filled with zeros). Rows whose words are not 4-byte aligned (K / 128 no multiple of 4) go through
    // registers, five aligned words for 16 K-blocks of a row: a load touches 32 rows, so it is the number
    // of loads that counts, and byte by byte they held 512 x 4096 x 11008 at 27 us. An image spans 16 K-blocks because handing one
    // over (copies in flight, the proxy fence, the arrival at the other CTA) takes 2,000 cycles, more
    // than four K-blocks' MMAs.
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = tile0; ok && t < tiles; t += tstep) {
      int mt, nt;
      tile_at(p, t, mt, nt);
      // This lane's rows: the weight blocks', then x's. A row past the matrix or the tile takes the last
      // one's scales: its operand is zero or no part of the MMA, and its output is not stored.
      const uint8_t* row[MT + kXRows];
#pragma unroll
      for (int b = 0; b < MT; ++b) {
        const int src = weight_source<MODE, CG>(pair, b);
        row[b] = p.ws[src] + min(weight_block<MODE, MT, CG>(nt, pair, b), (p.N - 1) / 128) * p.ldws[src];
      }
#pragma unroll
      for (int j = 0; j < kXRows; ++j) row[MT + j] = p.xs + min(mt * p.bn + j * 32 + lane, p.M - 1) * p.ldxs;
      for (int kb = kb0; kb < kb1; kb += kSfSpan) {
        if (!warp_all(mbar_poll(&sf_empty[s], ph ^ 1))) {
          ok = false;
          break;
        }
        uint8_t* im = smem + p.sf_off + s * (4 * sf_quad) + lane * 16;
        const int end = min(kb1, kb + kSfSpan);
        if (p.sf_words) {
          for (int kq = kb; kq < end; kq += 4, im += sf_quad) {
            const int left = min(4, p.kblocks - kq);
#pragma unroll
            for (int i = 0; i < MT + kXRows; ++i) {
              if (CG == 1 ? i >= MT && (i - MT) * 32 >= p.bn : i >= MT + 4 && sfb_groups == 1) break;
#pragma unroll
              for (int j = 0; j < (i < MT ? 4 : 1); ++j)
                scale_copy(im + scale_place(MT, i) + (i < MT ? 4 * j : 0), row[i] + kq, left);
            }
          }
        } else {
          auto stop = [&](int i) {  // the end of the matrix that row i is of
            const int src = weight_source<MODE, CG>(pair, i);
            return (i < MT ? p.ws[src] + (p.N - 1) / 128 * p.ldws[src] : p.xs + (p.M - 1) * p.ldxs) + p.kblocks;
          };
          auto place = [&](int i, const uint32_t (&w)[5]) {
            const uint32_t sh = 8 * (uint32_t)(reinterpret_cast<uintptr_t>(row[i] + kb) & 3);
#pragma unroll
            for (int q = 0; q < kSfSpan / 4; ++q) {
              const uint32_t v = __funnelshift_r(w[q], w[q + 1], sh);
              uint8_t* at = im + q * sf_quad + scale_place(MT, i);
              if (i < MT) *reinterpret_cast<uint4*>(at) = make_uint4(v, v, v, v);
              else *reinterpret_cast<uint32_t*>(at) = v;
            }
          };
          if constexpr (CG == 1) {  // few rows, and few registers: one row after the other
#pragma unroll
            for (int i = 0; i < MT + kXRows; ++i) {
              if (i >= MT && (i - MT) * 32 >= p.bn) break;
              uint32_t w[5];
              const bool cut = scale_words5(row[i] + kb, stop(i), w);
              if (__any_sync(0xffffffffu, cut)) scale_last_bytes(row[i] + kb, stop(i), w);
              place(i, w);
            }
          } else {
            uint32_t w[MT + kXRows][5];
            bool cut = false;
#pragma unroll
            for (int i = 0; i < MT + kXRows; ++i) cut |= scale_words5(row[i] + kb, stop(i), w[i]);
            if (__any_sync(0xffffffffu, cut)) {
#pragma unroll
              for (int i = 0; i < MT + kXRows; ++i) scale_last_bytes(row[i] + kb, stop(i), w[i]);
            }
#pragma unroll
            for (int i = 0; i < MT + kXRows; ++i)
              if (i < MT + 4 || sfb_groups == 2) place(i, w[i]);
          }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();  // generic-proxy writes -> the tensor core's reads
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) mbar_arrive_cluster(cluster_addr(&sf_full[s], 0));
          else mbar_arrive(&sf_full[s]);
        }
        if (++s == kSfSlots) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    for (int i = 0; i < kSfSlots && warp_all(mbar_poll(&sf_empty[s], ph ^ 1)); ++i)  // as the producer
      if (++s == kSfSlots) {
        s = 0;
        ph ^= 1;
      }
  } else if (warp == MW) {
    // ------------------------------------------------------------ MMA issuer
    // The tensor core's queue holds little more than the MMA it works on, so what this warp does between
    // two K-blocks has to fit beside the last MMAs of the first: descriptors advance by additions, and a
    // K tail costs no branch (the TMA's zeros fill it).
    if (pair == 0) {
      int s = 0, acc = 0, ss = 0;
      uint32_t ph = 0, aph = 0, sph = 0, sfbuf = 0;
      bool ok = true, issued = false;
      const uint32_t sf_cols = 4 * (MT + sfb_groups), sf_base = tmem + p.nacc * p.acc_cols;
      const uint32_t dstep = (uint32_t)p.stage_bytes >> 4;  // descriptors count in 16 bytes
      const uint64_t ad0 = umma_desc_sw128(smem_u32(smem));
      uint64_t ad = ad0;
      bool ready = false;
      constexpr uint32_t kNextScale = (1u << 29) | (1u << 4);  // the next byte of both scale words
      for (int t = tile0; ok && t < tiles; t += tstep) {
        if (!warp_all(mbar_wait_cg<CG>(&acc_empty[acc], aph ^ 1))) break;
        tc_fence_after();
        const uint32_t d0 = tmem + acc * p.acc_cols;
        uint32_t accumulate = 0;
        for (int kb = kb0; ok && kb < kb1; kb += kSfSpan) {
          if (!warp_all(mbar_wait_cg<CG>(&sf_full[ss], sph))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int end = min(kb1, kb + kSfSpan);
          uint32_t im = smem_u32(smem + p.sf_off) + ss * (4 * sf_quad);
          for (int kq = kb; ok && kq < end; kq += 4, im += sf_quad) {
            const uint32_t sf = sf_base + sfbuf * sf_cols;  // two sets of columns in turn
            if (elect_one())
              for (int g = 0; g < MT + sfb_groups; ++g) tmem_cp_scales<CG>(sf + 4 * g, im + g * kSfAtom);
            sfbuf ^= 1;
            uint32_t idesc = p.idesc;
            const int n = min(4, end - kq);
            for (int i = 0; i < n; i += KS) {
              if (!ready && !warp_all(mbar_poll(&full[s], ph))) {
                ok = false;
                break;
              }
              tc_fence_after();
              const int s1 = s + 1 == S ? 0 : s + 1;
              const bool next = mbar_test(&full[s1], ph ^ (s1 == 0 ? 1u : 0u));  // looked at while the MMAs are issued
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                  if (i + k >= n) break;
                  const uint64_t a = ad + k * (uint32_t)(block_bytes >> 4), bd = a + MT * (kGemmABlock >> 4);
#pragma unroll
                  for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int b = 0; b < MT; ++b)
                      umma_mxf8<CG>(d0 + b * p.bn, a + b * (kGemmABlock >> 4) + 2 * j, bd + 2 * j, idesc + k * kNextScale, sf + 4 * b,
                                    sf + 4 * MT, j || k ? 1u : accumulate);
                }
                umma_commit_cg<CG>(&empty[s]);
              }
              ready = warp_all(next);
              idesc += KS * kNextScale;
              accumulate = 1;
              issued = true;
              ad += dstep;
              s = s1;
              if (s == 0) {
                ph ^= 1;
                ad = ad0;
              }
            }
          }
          if (elect_one()) umma_commit_cg<CG>(&sf_empty[ss]);
          if (++ss == kSfSlots) {
            ss = 0;
            sph ^= 1;
          }
        }
        if (!ok) break;
        if (elect_one()) umma_commit_cg<CG>(&acc_full[acc]);
        if (++acc == p.nacc) {
          acc = 0;
          aph ^= 1;
        }
      }
      if (issued) {
        if (elect_one()) umma_commit_cg<CG>(done);  // every MMA this CTA issued has finished before TMEM is released
        mbar_settle(done, 0);
      }
    } else {
      mbar_settle(done, 0);  // the leader's commit arrives in both CTAs: the last signal that this one gets
    }
  } else if constexpr (CG == 2) {
    // ------------------------------------------------------------ epilogue
    // A lane holds one output n of a run of tokens, a warp 32 outputs and a group of four warps 128, and
    // each token's outputs are stored as one run; the two groups take alternate runs of tokens. The
    // accumulator is handed back once its last columns are in registers. After a wait that gave up
    // every warp runs on without work: all reach every barrier.
    const int q = warp & 3, g = warp >> 2;
    int acc = 0;
    uint32_t aph = 0;
    bool ok = true;
    auto release = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(cluster_addr(&acc_empty[acc], 0));
    };
    if constexpr (MODE == FP8_LINEAR) {
      const int nch = (p.bn + 31) / 32, items = MT * nch;
      for (int t = tile0; t < tiles; t += tstep) {
        ok = mbar_poll(&acc_full[acc], aph) && ok;
        tc_fence_after();
        int mt, nt;
        tile_at(p, t, mt, nt);
        const uint32_t base = tmem + acc * p.acc_cols + ((uint32_t)(q * 32) << 16);
        if (g >= items) release();
        for (int i = g; i < items; i += kFp8Epi / 4) {
          const int blk = i / nch, c = (i - blk * nch) * 32;  // bn is a multiple of 32
          const int n = weight_block<MODE, MT, CG>(nt, pair, blk) * 128 + q * 32 + lane;
          const int m0 = mt * p.bn + c;
          const int cols = ok ? min(32, p.M - m0) : 0;  // tokens of this run
          uint32_t v[32];
          tmem_ld16(base + blk * p.bn + c, reinterpret_cast<uint32_t(&)[16]>(v[0]));
          tmem_ld16(base + blk * p.bn + c + 16, reinterpret_cast<uint32_t(&)[16]>(v[16]));
          tmem_ld_wait();
          if (i + kFp8Epi / 4 >= items) release();
          if (n < p.N) {
            if (p.out_type == FT_BF16) store_columns(static_cast<__nv_bfloat16*>(p.out), p.ldo, v, n, m0, cols);
            else if (p.out_type == FT_F16) store_columns(static_cast<__half*>(p.out), p.ldo, v, n, m0, cols);
            else store_columns(static_cast<float*>(p.out), p.ldo, v, n, m0, cols);
          }
        }
        if (++acc == p.nacc) {
          acc = 0;
          aph ^= 1;
        }
      }
    } else {
      // Of each two runs of 16 tokens the leader finishes the first and the other CTA the second: a warp sends
      // the peer's warp of the same lanes its product's columns of the peer's run, and takes the peer's
      // columns of its own run. Two buffers, and no message that says one is free: a warp sends run k
      // only after it has used the peer's run k - 1, which the peer sent after it had used this
      // warp's run k - 2. (With releases in place of st.async each exchange waited for the rounded
      // values' global stores: 23,000 cycles per tile of 224 tokens.)
      uint8_t* recv = smem + p.stg_off + warp * (2 * kFp8WarpSwap) + lane * 16;  // [4 tokens each][lane][4]
      float* tops = reinterpret_cast<float*>(smem + p.stg_off + kFp8SwapBytes) + g * (2 * kFp8Chunk * 4);
      uint64_t* swap = reinterpret_cast<uint64_t*>(smem + p.bar_off + kFp8SwapBar) + 2 * warp;  // the peer's columns have come
      const uint32_t peer_recv = cluster_addr(recv, 1 - pair), peer_swap = cluster_addr(swap, 1 - pair);
      const int pairs = p.bn / (2 * kFp8Chunk);
      int sbuf = 0, rbuf = 0;
      uint32_t rph = 0;
      for (int t = tile0; t < tiles; t += tstep) {
        ok = mbar_poll(&acc_full[acc], aph) && ok;
        tc_fence_after();
        int mt, nt;
        tile_at(p, t, mt, nt);
        const uint32_t base = tmem + acc * p.acc_cols + ((uint32_t)(q * 32) << 16);
        const int n = nt * 128 + q * 32 + lane;
        auto send = [&](int i) {
          uint32_t u[kFp8Chunk];
          tmem_ld16(base + i * 2 * kFp8Chunk + (1 - pair) * kFp8Chunk, u);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < kFp8Chunk; e += 4) st_async4(peer_recv + sbuf * kFp8WarpSwap + e * (32 * 4), u + e, peer_swap + 8 * sbuf);
          sbuf ^= 1;
        };
        if (g >= pairs) release();
        else send(g);
        for (int i = g; i < pairs; i += kFp8Epi / 4) {
          uint32_t v[kFp8Chunk], u[kFp8Chunk];
          tmem_ld16(base + i * 2 * kFp8Chunk + pair * kFp8Chunk, v);
          if (lane == 0) mbar_arrive_expect_tx(&swap[rbuf], kFp8WarpSwap);
          ok = mbar_settle<true>(&swap[rbuf], rph) && ok;  // the peer sends every run, after a wait that gave up too
#pragma unroll
          for (int e = 0; e < kFp8Chunk; e += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(recv + rbuf * kFp8WarpSwap + e * (32 * 4));
            u[e] = w.x;
            u[e + 1] = w.y;
            u[e + 2] = w.z;
            u[e + 3] = w.w;
          }
          tmem_ld_wait();
          const int m0 = mt * p.bn + i * 2 * kFp8Chunk + pair * kFp8Chunk, cols = ok ? min(kFp8Chunk, p.M - m0) : 0;
          float* part = tops + rbuf * (kFp8Chunk * 4);
          auto next = [&] {
            if (i + kFp8Epi / 4 < pairs) send(i + kFp8Epi / 4);
            else release();
          };
          if (pair == 0) swiglu_columns(p, v, u, n, m0, cols, part, 1 + g, q, lane, next);
          else swiglu_columns(p, u, v, n, m0, cols, part, 1 + g, q, lane, next);
          rbuf ^= 1;
          if (rbuf == 0) rph ^= 1;
        }
        if (++acc == p.nacc) {
          acc = 0;
          aph ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ this rank's part of a tile
    const int q = warp & 3, g = warp >> 2;
    float* red = reinterpret_cast<float*>(smem);  // [MT * bn][128] over the stages, which every MMA has read
    part_ok = mbar_poll(&acc_full[0], 0);
    if (part_ok) {
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
  if constexpr (CG == 1) {
    // The parts are added in rank order; each rank finishes every split-th run of eight tokens, a warp
    // a token (128 outputs, four per lane).
    cluster_sync();
    if (warp < kFp8Epi && part_ok) {
      int mt, nt;
      tile_at(p, tile0, mt, nt);
      for (int c = rank * kFp8Epi + warp; c < p.bn; c += p.split * kFp8Epi) {
        const int m = mt * p.bn + c;
        if (m >= p.M) break;
        float4 v[MT];
#pragma unroll
        for (int b = 0; b < MT; ++b) {
          v[b] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int r0 = 0; r0 < p.split; r0 += 4) {  // four loads in flight
            float4 part[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r0 + r < p.split) part[r] = ld_cluster_f4(cluster_addr(smem + ((b * p.bn + c) * 128 + lane * 4) * 4, r0 + r));
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r0 + r < p.split) {
                v[b].x += part[r].x;
                v[b].y += part[r].y;
                v[b].z += part[r].z;
                v[b].w += part[r].w;
              }
          }
        }
        if constexpr (MODE == FP8_SWIGLU) finish_swiglu(p, m, nt * 128 + lane * 4, v[0], v[1]);
        else finish_linear(p, m, nt * 128 + lane * 4, v[0]);
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  // No CTA leaves while another reads its shared memory (parts of a tile), or before the arrivals that the other
  // one's threads made at it (they come before those threads' arrival here). What comes on its own, tcgen05.commit,
  // copies and st.async, has been waited for: the barrier says nothing about it.
  cluster_sync();
  tc_fence_after();
  if (warp == MW) tmem_dealloc_cg<CG>(tmem, p.tmem_cols);
}

}  // namespace ixb
