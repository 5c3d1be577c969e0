// MXFP4 quantize / unpack kernels (HBM-bound) and the block helpers the
// MXFP4 GEMM epilogues share.
//
// Per block of 32 consecutive values of a row (the OCP microscaling format):
//   e    = floor(log2(max |x|)) - 2, clamped to >= -127; byte s = e + 127
//   code = e2m1_rne_sat(x * 2^-e), sign from x
//   a block with an infinity or a NaN: s = 0xFF (NaN), codes 0
// 2^-e is a power of two, so x * 2^-e is exact and the only rounding is the
// E2M1 one.  There is no tensor-wide scale and therefore no amax pass: one
// read of x and one write of the codes and scales.  32768 x 14336 bf16 there and
// back, calls in a row: 364 us, 6.5 TB/s (a launch of either kernel alone takes
// 177 us, some of its writes still in L2 when it ends).
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

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

// Loads of what an earlier launch may still be writing while this one starts:
// ordinary ones (the read-only path wants data that never changes under it).
__device__ __forceinline__ uint4 ld_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// ---------------------------------------------------------------- typed 8-value loads / stores
template <typename T>
struct Vec8;                       // 8 values of T as 16-byte words
template <>
struct Vec8<__nv_bfloat16> {
  uint4 w;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { w = ld_v4(p); }
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
  __device__ __forceinline__ void load(const __half* p) { w = ld_v4(p); }
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

// ---------------------------------------------------------------- wide accesses
// 32 bytes per lane in one access (256-bit, 32-byte aligned): a warp moves 1 KiB
// of one row, whole sectors each.
__device__ __forceinline__ void ld_v8(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
__device__ __forceinline__ void st_v8(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// VPL values of T per lane: 8 by 16-byte accesses, 16 by 32-byte ones.
template <typename T, int VPL>
struct Lane {
  static constexpr int WORDS = VPL * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const T* p) {
    const char* c = reinterpret_cast<const char*>(p);
    if constexpr (VPL == 16) {
#pragma unroll
      for (int i = 0; i < WORDS / 8; ++i)
        ld_v8(c + i * 32, *reinterpret_cast<uint32_t(*)[8]>(w + i * 8));
    } else {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i)
        *reinterpret_cast<uint4*>(w + i * 4) = ld_v4(c + i * 16);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    char* c = reinterpret_cast<char*>(p);
    if constexpr (VPL == 16) {
#pragma unroll
      for (int i = 0; i < WORDS / 8; ++i)
        st_v8(c + i * 32, *reinterpret_cast<const uint32_t(*)[8]>(w + i * 8));
    } else {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i)
        *reinterpret_cast<uint4*>(c + i * 16) = *reinterpret_cast<const uint4*>(w + i * 4);
    }
  }
  __device__ __forceinline__ float2 get2(int i) const {      // values 2 i and 2 i + 1
    if constexpr (std::is_same<T, float>::value)
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (std::is_same<T, __half>::value)
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    else
      return bf16x2_to_f2(w[i]);
  }
  __device__ __forceinline__ void set2(int i, float a, float b) {
    if constexpr (std::is_same<T, float>::value) {
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    } else {
      w[i] = pack2(a, b, T());
    }
  }
  // max |v| as fp32 bits; 16-bit values compare as their magnitudes' integers,
  // two at a time (a NaN's are above every number's)
  __device__ __forceinline__ uint32_t absmax_bits() const {
    uint32_t m = 0;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
      m = max(m & 0xFFFFu, m >> 16);
      if constexpr (std::is_same<T, __half>::value)
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
      return m << 16;
    }
  }
};

// ---------------------------------------------------------------- quantize
constexpr int kThreads = 256;

// A warp's unit of work is UNROLL * 32 * VPL consecutive values of a row (units
// grid-stride over rows and pieces alike, so one long row spreads over many
// warps): 32 / VPL lanes per block, UNROLL loads in flight per lane.  The four
// scales of a 128-value stretch are neighbours in the blocked layout and leave
// as one word.  Scales of rows in [M, Mpad) and of the columns that pad a row's
// last tile are written as 0.
template <typename T, int VPL, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    k_mxfp4_quantize(const T* x, int64_t M, int64_t K, int64_t ldx, uint8_t* q, int64_t ldq,
                     uint8_t* sf, int64_t Mpad, uint32_t units_per_row) {
  grid_wait();
  grid_launch_dependents();
  constexpr int LPB = BLOCK / VPL;                 // lanes per block
  const int lane = threadIdx.x & 31;
  const int k = (int)K;
  const int64_t c4 = sf_tiles(K);
  const int padded = (int)(c4 * 128);              // values up to the padded width
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t units = Mpad * units_per_row;
  for (int64_t wi = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); wi < units;
       wi += warps) {
    const int64_t r = wi / units_per_row;
    const int v0 = (int)(wi - r * units_per_row) * (32 * VPL * UNROLL) + lane * VPL;
    const bool real = r < M;
    const T* xr = x + r * ldx;
    uint8_t* qr = q + r * ldq;
    uint8_t* sr = sf + sf_swizzled_offset(r, 0, c4);
    Lane<T, VPL> raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int v = v0 + u * 32 * VPL;
      raw[u].zero();
      if (real && v < k) raw[u].load(xr + v);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int v = v0 + u * 32 * VPL;
      uint32_t m = raw[u].absmax_bits();
#pragma unroll
      for (int o = 1; o < LPB; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t s = scale_byte(m);
      const float inv = scale_inverse(s);
      uint32_t code[VPL / 8];
#pragma unroll
      for (int c = 0; c < VPL / 8; ++c) {
        code[c] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = raw[u].get2(c * 4 + i);
          float a, b;
          mul_rn_f32x2(f.x, f.y, inv, a, b);
          code[c] |= f32x2_to_e2m1x2(a, b) << (8 * i);
        }
        if (inv == 0.f) code[c] = 0u;              // a NaN block
      }
      uint32_t word = s | __shfl_down_sync(0xffffffffu, s, LPB) << 8;
      word |= __shfl_down_sync(0xffffffffu, word, 2 * LPB) << 16;
      if (real && v < k) {
        if constexpr (VPL == 16)
          *reinterpret_cast<uint2*>(qr + (v >> 1)) = make_uint2(code[0], code[1]);
        else
          *reinterpret_cast<uint32_t*>(qr + (v >> 1)) = code[0];
      }
      if (lane % (4 * LPB) == 0 && v < padded)
        *reinterpret_cast<uint32_t*>(sr + (int64_t)(v >> 7) * 512) = word;
    }
  }
}

// ---------------------------------------------------------------- unpack
// Units as in the quantizer: a lane turns VPL codes into VPL values of T.
template <typename T, int VPL, int UNROLL>
__global__ void __launch_bounds__(kThreads)
    k_mxfp4_dequantize(const uint8_t* q, const uint8_t* sf, int64_t M, int64_t K, T* out,
                       int64_t ldo, uint32_t units_per_row) {
  grid_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int k = (int)K;
  const int64_t c4 = sf_tiles(K);
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  const int64_t units = M * units_per_row;
  for (int64_t wi = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); wi < units;
       wi += warps) {
    const int64_t r = wi / units_per_row;
    const int v0 = (int)(wi - r * units_per_row) * (32 * VPL * UNROLL) + lane * VPL;
    const uint8_t* qr = q + r * (K >> 1);
    const uint8_t* sr = sf + sf_swizzled_offset(r, 0, c4);
    T* orow = out + r * ldo;
    uint32_t code[UNROLL][VPL / 8];
    uint8_t s[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int v = v0 + u * 32 * VPL;
      if (v < k) {
        if constexpr (VPL == 16) {
          const uint2 c = *reinterpret_cast<const uint2*>(qr + (v >> 1));
          code[u][0] = c.x;
          code[u][1] = c.y;
        } else {
          code[u][0] = *reinterpret_cast<const uint32_t*>(qr + (v >> 1));
        }
        s[u] = sr[(int64_t)(v >> 7) * 512 + ((v >> 5) & 3)];
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int v = v0 + u * 32 * VPL;
      if (v >= k) break;
      const float sc = scale_value(s[u]);
      Lane<T, VPL> o;
#pragma unroll
      for (int c = 0; c < VPL / 8; ++c) {
        uint32_t hx2[4];
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
            : "=r"(hx2[0]), "=r"(hx2[1]), "=r"(hx2[2]), "=r"(hx2[3])
            : "r"(code[u][c]));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // exact in fp32: one significant bit more than the scale's
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hx2[i]));
          o.set2(c * 4 + i, f.x * sc, f.y * sc);
        }
      }
      o.store(orow + v);
    }
  }
}

}  // namespace mx
}  // namespace h3b
