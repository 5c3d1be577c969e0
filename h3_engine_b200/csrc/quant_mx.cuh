// MXFP4 quantize / unpack kernels (HBM-bound) and the block helpers the
// MXFP4 GEMM epilogues share.
//
// Per block of 32 consecutive values of a row (the OCP microscaling format):
//   e    = floor(log2(max |x|)) - 2, clamped to >= -127; byte s = e + 127
//   code = e2m1_rne_sat(x * 2^-e), sign from x
//   a block with an infinity or a NaN: s = 0xFF (NaN), codes 0
// 2^-e is a power of two, so x * 2^-e is exact and the only rounding is the
// E2M1 one.  There is no tensor-wide scale and therefore no amax pass: one
// read of x and one write of the codes and scales.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "quant.cuh"

namespace h3b {
namespace mx {

constexpr int BLOCK = 32;

// Bytes of a row's blocked scales are padded to whole 128 x 4 tiles.
__host__ __device__ __forceinline__ int64_t sf_tiles(int64_t k) { return (k / BLOCK + 3) >> 2; }

// Byte of the shared scale from the bits of max |x| (fp32): exponent field - 2,
// not below 0 (2^-127, which also covers zeros and subnormals); 0xFF when the
// block holds a non-finite value.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^-(s - 127) for a byte from scale_byte (s <= 252: always a normal number);
// 0 for the NaN scale, whose codes are 0.
__device__ __forceinline__ float scale_inverse(uint32_t s) {
  return s == 255u ? 0.f : __uint_as_float((254u - s) << 23);
}
// 2^(s - 127); s = 0 is the subnormal 2^-127, s = 255 NaN.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return s == 0u ? __uint_as_float(0x00400000u)
                 : (s == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(s << 23));
}

// Four code bytes of 8 values.  A non-finite value times inv = 0 is NaN, whose
// conversion is not a zero code: the caller clears the codes of such a block.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float inv) {
  uint32_t packed = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    mul_rn_f32x2(v[2 * i], v[2 * i + 1], inv, a, b);
    packed |= f32x2_to_e2m1x2(a, b) << (8 * i);
  }
  return inv != 0.f ? packed : 0u;
}

// ---------------------------------------------------------------- typed 8-value loads / stores
template <typename T>
struct Vec8;                       // 8 values of T as 16-byte words
template <>
struct Vec8<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = ld_nc_v4(p); }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Vec8<__half> {
  uint4 w;
  __device__ __forceinline__ void load(const __half* p) { w = ld_nc_v4(p); }
  __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Vec8<float> {
  uint4 w[2];
  __device__ __forceinline__ void load(const float* p) {
    w[0] = ld_nc_v4(p);
    w[1] = ld_nc_v4(p + 4);
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(w[i].x);
      v[4 * i + 1] = __uint_as_float(w[i].y);
      v[4 * i + 2] = __uint_as_float(w[i].z);
      v[4 * i + 3] = __uint_as_float(w[i].w);
    }
  }
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// max |v| of 8 values as fp32 bits (a NaN's bits are above every number's)
__device__ __forceinline__ uint32_t absmax_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// Lets the next launch of the stream start before this one is done, where that
// launch waits for this one before it reads its results.
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Waits until the launch before this one is done and its results are visible
// (at once, where this one was not started early).
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- quantize
constexpr int kThreads = 256;

// A warp's unit of work is UNROLL * 256 consecutive values of a row (units
// grid-stride over rows and pieces alike, so one long row spreads over many
// warps): four lanes per 32-value block, each lane 8 values per step, UNROLL
// loads in flight.  Scales of rows in [M, Mpad) and of the columns that pad a
// row's last tile are written as 0.
template <typename T, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    k_mxfp4_quantize(const T* __restrict__ x, int64_t M, int64_t K, int64_t ldx,
                     uint8_t* __restrict__ q, uint8_t* __restrict__ sf, int64_t Mpad,
                     uint32_t units_per_row, int early) {
  if (early) grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int steps = (int)(K >> 3);                 // 8-value pieces of a row
  const int64_t c4 = sf_tiles(K);
  const int padded = (int)(c4 * 16);               // pieces up to the padded width
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t units = Mpad * units_per_row;
  for (int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < units;
       w += warps) {
    const int64_t r = w / units_per_row;
    const int h0 = (int)(w - r * units_per_row) * (32 * UNROLL);
    const bool real = r < M;
    const T* xr = x + r * ldx;
    uint8_t* qr = q + r * (K >> 1);
    Vec8<T> raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * 32 + lane;
      raw[u].zero();
      if (real && h < steps) raw[u].load(xr + (int64_t)h * 8);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * 32 + lane;
      float v[8];
      raw[u].get(v);
      uint32_t m = absmax_bits8(v);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t s = scale_byte(m);
      if (real && h < steps)
        *reinterpret_cast<uint32_t*>(qr + (int64_t)h * 4) = codes8(v, scale_inverse(s));
      if ((lane & 3) == 0 && h < padded)
        sf[sf_swizzled_offset(r, h >> 2, c4)] = static_cast<uint8_t>(s);
    }
  }
}

// ---------------------------------------------------------------- unpack
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                            pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2(v[0], v[1], __half()), pack2(v[2], v[3], __half()),
                 pack2(v[4], v[5], __half()), pack2(v[6], v[7], __half()));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// 8 E2M1 codes (4 bytes) times a scale, in fp32 (exact: one significant bit
// more than the scale's).
__device__ __forceinline__ void values8(uint32_t codes, float s, float (&v)[8]) {
  uint32_t hx2[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(hx2[0]), "=r"(hx2[1]), "=r"(hx2[2]), "=r"(hx2[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hx2[i]));
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
}

// Units of UNROLL * 256 values as in the quantizer: lane l takes the 8-value
// pieces l, l + 32, ... of the unit, all loads in flight.
template <typename T, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    k_mxfp4_dequantize(const uint8_t* __restrict__ q, const uint8_t* __restrict__ sf, int64_t M,
                       int64_t K, T* __restrict__ out, int64_t ldo, uint32_t units_per_row) {
  const int lane = threadIdx.x & 31;
  const int steps = (int)(K >> 3);
  const int64_t c4 = sf_tiles(K);
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t units = M * units_per_row;
  for (int64_t w = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); w < units;
       w += warps) {
    const int64_t r = w / units_per_row;
    const int h0 = (int)(w - r * units_per_row) * (32 * UNROLL) + lane;
    const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + r * (K >> 1));
    T* orow = out + r * ldo;
    uint32_t codes[UNROLL];
    uint8_t s[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * 32;
      codes[u] = 0;
      s[u] = 0;
      if (h < steps) {
        codes[u] = __ldg(qr + h);
        s[u] = __ldg(sf + sf_swizzled_offset(r, h >> 2, c4));
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * 32;
      if (h >= steps) break;
      float v[8];
      values8(codes[u], scale_value(s[u]), v);
      store8(orow + (int64_t)h * 8, v);
    }
  }
}

}  // namespace mx
}  // namespace h3b
