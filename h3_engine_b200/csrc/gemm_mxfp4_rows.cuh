// MXFP4 product for few rows of activations (single tokens, text and
// conditioning rows), where reading the weight once is the bound: up to 128, or a
// few tiles of 128.
//
// The operands change places: the weight's 128-row tiles are the MMA's M side
// and the MT (16 ... 128) activation rows its N side, so every byte that
// streams in is weight (the 128-row activation tile of the large kernel would
// be almost empty).  D^T lies in TMEM with weight rows as lanes, and a warp's
// 32 lanes are 32 consecutive output columns.
//
// There are few weight tiles (N / 128), so a cluster of CTAs splits K: each
// computes a partial D^T of its k-blocks, leaves it in its shared memory, and
// the CTAs then each add up a share of the rows over distributed shared memory,
// always in rank order, and run the epilogue.  Two CTAs fit an SM, and a CTA's
// share of K usually fits its ring, so the whole weight is in flight at once.
// 1 x 7168 x 5376 (20.5 MB): 6.9 us, 3 TB/s, the rest of it the launch, the first
// loads' latency and the cluster's two barriers.
//
// Inside one entry point's chain of launches (quantize, product, or quantize,
// up, down) the weight's loads do not depend on the launch before, which only
// produces the activation's codes: there the kernel fills its ring before it
// waits for that launch.
#pragma once

#include "gemm_mxfp4.cuh"

namespace h3b {
namespace mxrows {

using mxgemm::KB_ATOMS;
using mxgemm::KB_BYTES;
using mxgemm::KB_ELEMS;
using mxgemm::SF_ATOM;

constexpr int BN = 128;                       // weight rows per tile
constexpr int THREADS = 192;                  // producer, MMA, 4 epilogue warps
constexpr int kMaxRows = 128;                 // of one tile
constexpr int kFusedRows = 32;                // rows that the kernel can quantize itself,
constexpr int kUnitRows = 8;                  // in units of 8 rows of a k-block
constexpr int kMaxSplit = 8;
constexpr uint32_t TMEM_COLS = 256;           // two CTAs per SM
constexpr uint32_t SF_COL = 128;
constexpr uint32_t SF_STAGE_COLS = 2 * KB_ATOMS * 4;

template <int MT>
struct Ring {
  static constexpr int W_BYTES = BN * KB_BYTES;
  static constexpr int X_BYTES = MT * KB_BYTES;
  static constexpr int SF_BYTES = KB_ATOMS * SF_ATOM;       // of the weight, and of the rows
  static constexpr int STAGE = W_BYTES + X_BYTES + 2 * SF_BYTES;
  static constexpr int STAGES = MT <= 32 ? 5 : (MT == 64 ? 4 : 3);
  static constexpr int BAR_OFF = STAGES * STAGE;
  static constexpr int BYTES = BAR_OFF + 128 + 1024;
  static_assert(STAGE % 1024 == 0, "swizzle alignment");
  static_assert(MT * BN * 4 <= STAGES * STAGE, "the partial product reuses the ring");
  static_assert(2 * (BYTES + 1024) <= 233472, "two CTAs per SM");
  static_assert(SF_COL + STAGES * SF_STAGE_COLS <= TMEM_COLS, "TMEM budget");
};

struct Args {
  CUtensorMap tmap_w;      // u8 [N, K/2], box 128 B x 128 rows, 128B swizzle
  CUtensorMap tmap_x;      // u8 [M, K/2], box 128 B x MT rows, 128B swizzle (not FUSED)
  const uint8_t* sfw;
  const uint8_t* sfx;      // not FUSED
  const void* x;           // FUSED: [M, K], row stride ldx
  long long ldx;
  const void* bias;
  const void* residual;
  void* out;
  uint8_t* q_out;          // kSwigluQuant: codes u8 [M, N/4] and blocked scales
  uint8_t* sf_out;
  long long ldr, ldd;
  int M, N, K;
  int sf_tiles_k;
  int act;
  int first;               // of a call: the weight, too, follows the launches before
};

// Four consecutive 16-bit values.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = mxgemm::unpack2(w.x, T()), b = mxgemm::unpack2(w.y, T());
  return make_float4(a.x, a.y, b.x, b.y);
}

// Two MMA k-steps under one elected lane: the scale tiles of the weight rows
// and of the activation rows, then one or two MMAs.
template <int MT>
__device__ __forceinline__ void kpair_elect(uint32_t sfw_t, uint64_t sfw_d, uint32_t sfx_t,
                                            uint64_t sfx_d, uint32_t d_tmem, uint64_t w_desc,
                                            uint64_t x_desc, uint32_t accumulate,
                                            uint32_t second) {
  asm volatile(
      "{\n\t.reg .pred p, e, f;\n\t"
      "setp.ne.b32 p, %7, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t"
      "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%2], %3;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X"
      " [%4], %5, %6, %8, [%0], [%2], p;\n\t"
      "setp.ne.and.b32 f, %10, 0, e;\n\t"
      "setp.eq.u32 p, 0, 0;\n\t"
      "@f tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X"
      " [%4], %11, %12, %9, [%0], [%2], p;\n\t}" ::"r"(sfw_t),
      "l"(sfw_d), "r"(sfx_t), "l"(sfx_d), "r"(d_tmem), "l"(w_desc), "l"(x_desc), "r"(accumulate),
      "r"(mxgemm::idesc(BN, MT, 0)), "r"(mxgemm::idesc(BN, MT, 2)), "r"(second), "l"(w_desc + 2),
      "l"(x_desc + 2)
      : "memory");
}

// Warp-collective load of NC consecutive 32-bit TMEM columns (a multiple of 16).
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
// Cluster barrier without ordering earlier memory operations.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::
                   : "memory");
}
// Sum over the cluster, in rank order, of the float4 at `addr`; all loads are
// in flight together.
__device__ __forceinline__ float4 cluster_sum(uint32_t addr, int ranks) {
  float4 v[kMaxSplit];
#pragma unroll
  for (int c = 0; c < kMaxSplit; ++c)
    v[c] = c < ranks ? ld_cluster_f4(mapa_shared(addr, c)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 t = v[0];
#pragma unroll
  for (int c = 1; c < kMaxSplit; ++c)
    t = make_float4(t.x + v[c].x, t.y + v[c].y, t.z + v[c].z, t.w + v[c].w);
  return t;
}

// FUSED: the activation arrives as 16-bit rows and the epilogue warps quantize
// it into the ring themselves, units of 8 rows of a k-block in turn (1: there are
// 8 rows at most).
template <int MT, typename T, int EPI, int FUSED>
__global__ void __launch_bounds__(THREADS) k_gemm_mxfp4_rows(const __grid_constant__ Args p) {
  using R = Ring<MT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + R::BAR_OFF);
  uint64_t* full = bars;
  uint64_t* empty = bars + R::STAGES;
  uint64_t* acc_full = bars + 2 * R::STAGES;
  uint64_t* drain = bars + 2 * R::STAGES + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * R::STAGES + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ranks = (int)gridDim.x, rank = (int)blockIdx.x;   // the cluster spans grid x
  const int n0 = (int)blockIdx.y * BN;
  const int m0 = (int)blockIdx.z * MT;         // first row of this tile of activations
  const int rows = min(MT, p.M - m0);
  const int num_kb = (p.K + KB_ELEMS - 1) / KB_ELEMS;
  const int kb0 = (int)((long long)num_kb * rank / ranks);
  const int kb1 = (int)((long long)num_kb * (rank + 1) / ranks);

  auto sW = [&](int s) { return smem + s * R::STAGE; };
  auto sX = [&](int s) { return smem + s * R::STAGE + R::W_BYTES; };
  auto sSFW = [&](int s) { return smem + s * R::STAGE + R::W_BYTES + R::X_BYTES; };
  auto sSFX = [&](int s) { return sSFW(s) + R::SF_BYTES; };

  const int groups = FUSED == 1 ? 1 : (rows + kUnitRows - 1) / kUnitRows;

  if (threadIdx.x == 0) {
    for (int s = 0; s < R::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), FUSED ? 1 + groups : 1);   // the loads; the quantized rows
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(acc_full), 1);
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&]() {
    if (!*abort_flag) {
      record_error(H3B_ERR_TIMEOUT);
      *abort_flag = 1;
    }
  };

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&p.tmap_w);
      if (!FUSED) prefetch_tmap(&p.tmap_x);
      auto sf_bytes = [&](int kb) {
        return (uint32_t)min(KB_ATOMS, p.sf_tiles_k - kb * KB_ATOMS) * SF_ATOM;
      };
      const uint8_t* sfw = p.sfw + (size_t)blockIdx.y * p.sf_tiles_k * SF_ATOM;
      const uint8_t* sfx = p.sfx + (size_t)blockIdx.z * p.sf_tiles_k * SF_ATOM;   // z > 0: MT 128
      auto load_w = [&](int kb, int s) {
        const uint32_t fb = smem_u32(&full[s]);
        mbar_expect_tx(fb, R::W_BYTES + sf_bytes(kb) + (FUSED ? 0 : R::X_BYTES + sf_bytes(kb)));
        tma_load_2d(smem_u32(sW(s)), &p.tmap_w, kb * KB_BYTES, n0, fb);
        bulk_load(smem_u32(sSFW(s)), sfw + (size_t)kb * KB_ATOMS * SF_ATOM, sf_bytes(kb), fb);
      };
      auto load_x = [&](int kb, int s) {
        if (FUSED) return;
        const uint32_t fb = smem_u32(&full[s]);
        tma_load_2d(smem_u32(sX(s)), &p.tmap_x, kb * KB_BYTES, m0, fb);
        bulk_load(smem_u32(sSFX(s)), sfx + (size_t)kb * KB_ATOMS * SF_ATOM, sf_bytes(kb), fb);
      };
      if (p.first) grid_wait();
      const int n = kb1 - kb0, head = min(n, R::STAGES);
      for (int i = 0; i < head; ++i) load_w(kb0 + i, i);
      if (!FUSED) grid_wait();           // the activation's codes are there from here on
      for (int i = 0; i < head; ++i) load_x(kb0 + i, i);
      int issued = head;
      bool ok = true;
      for (int i = head; i < n; ++i) {
        const int s = i % R::STAGES;
        if (!mbar_wait(smem_u32(&empty[s]), ((i / R::STAGES) & 1) ^ 1, abort_flag)) {
          fail();
          ok = false;
          break;
        }
        load_w(kb0 + i, s);
        load_x(kb0 + i, s);
        ++issued;
      }
      if (!ok || *abort_flag) {
        // let every copy in flight land before the CTA can exit (a stage whose
        // rows never came only runs out its wait)
        for (int i = max(0, issued - R::STAGES); i < issued; ++i)
          mbar_wait(smem_u32(&full[i % R::STAGES]), (i / R::STAGES) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort_flag));
    };
    bool ok = true;
    for (int i = 0; i < kb1 - kb0; ++i) {
      const int s = i % R::STAGES, kb = kb0 + i;
      if (!wait(&full[s], (i / R::STAGES) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int steps = min(4, (p.K - kb * KB_ELEMS + 63) >> 6);
      const uint32_t sf_t = tmem + SF_COL + s * SF_STAGE_COLS;
      const uint64_t sfw_d = desc_sf_atom(smem_u32(sSFW(s)));
      const uint64_t sfx_d = desc_sf_atom(smem_u32(sSFX(s)));
      const uint64_t w_d = desc_kmajor_sw128(smem_u32(sW(s)));
      const uint64_t x_d = desc_kmajor_sw128(smem_u32(sX(s)));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h * 2 < steps)
          kpair_elect<MT>(sf_t + h * 4, sfw_d + ((h * SF_ATOM) >> 4), sf_t + 8 + h * 4,
                          sfx_d + ((h * SF_ATOM) >> 4), tmem, w_d + h * 4, x_d + h * 4,
                          (i | h) != 0, h * 2 + 1 < steps);
      }
      tc_commit_elect(smem_u32(&empty[s]));
    }
    if (ok) {
      tc_commit_elect(smem_u32(acc_full));
    } else {
      if (lane == 0) fail();
      tc_commit_elect(smem_u32(drain));
      mbar_wait(smem_u32(drain), 0, nullptr);
    }
  } else {
    grid_wait();                         // x, bias, residual and out follow earlier work
    if (FUSED) {
      // rows r0 .. r0 + 7 of k-block i: lane l holds values 8 l .. 8 l + 7 of a row
      for (int i = FUSED == 1 ? warp - 2 : 0, g = FUSED == 1 ? 0 : warp - 2;;) {
        for (; g >= groups; g -= groups) ++i;
        if (i >= kb1 - kb0) break;
        const int r0 = FUSED == 1 ? 0 : g * kUnitRows;
        const int s = i % R::STAGES, piece = (kb0 + i) * (KB_ELEMS / 8) + lane;
        const bool in_k = piece * 8 < p.K;
        const T* x = static_cast<const T*>(p.x) + (size_t)r0 * p.ldx + (size_t)piece * 8;
        mx::Vec8<T> raw[kUnitRows];
#pragma unroll
        for (int r = 0; r < kUnitRows; ++r) {
          raw[r].zero();
          if (r0 + r < p.M && in_k) raw[r].load(x + (size_t)r * p.ldx);
        }
        if (i >= R::STAGES &&
            !__all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[s]), ((i / R::STAGES) & 1) ^ 1,
                                               abort_flag))) {
          fail();
          break;
        }
        uint8_t* xs = sX(s) + r0 * 128;
        uint8_t* sf = sSFX(s) + (lane >> 4) * SF_ATOM + ((lane >> 2) & 3) + r0 * 16;
#pragma unroll
        for (int r = 0; r < kUnitRows; ++r) {
          if (r0 + r < p.M) {
            float v[8];
            raw[r].get(v);
            uint32_t m = mx::absmax_bits8(v);
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const uint32_t sb = mx::scale_byte(m);
            *reinterpret_cast<uint32_t*>(xs + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) +
                                         (lane & 3) * 4) = mx::codes8(v, mx::scale_inverse(sb));
            if (!(lane & 3)) sf[r * 16] = (uint8_t)sb;
          }
        }
        fence_proxy_async_smem();        // the MMA reads them through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full[s]));
        if (FUSED == 1) i += 4;
        else g += 4;
      }
    }
    grid_launch_dependents();
    // partial D^T of this CTA, row-major [MT][128], over the ring (every load
    // has landed and been read when the accumulator is complete)
    float* part = reinterpret_cast<float*>(smem);
    const int qd = warp & 3;
    const bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_full), 0, abort_flag));
    if (ready) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < MT; c += 16) {
        if (c < rows) {
          uint32_t acc[16];
          tmem_ld_x16(tmem + ((uint32_t)(qd * 32) << 16) + c, acc);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < rows) part[(c + i) * BN + qd * 32 + lane] = __uint_as_float(acc[i]);
        }
      }
    } else {
      fail();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  if (ranks > 1) cluster_sync_all();     // every CTA's partial is there
  const uint32_t base = smem_u32(smem);
  // (warps 0 and 1 have not waited for the chain's earlier launches: the
  // residual and out are theirs too)
  grid_wait();
  if (EPI == mxgemm::kOut) {
    // 32 threads cover a row's 128 columns, four each
    const int c = (threadIdx.x & 31) * 4, n = n0 + c;
    const T* residual = static_cast<const T*>(p.residual);
    if (n < p.N) {                       // N % 8 == 0: all four or none
      float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.bias) b = load4(static_cast<const T*>(p.bias) + n);
      for (int m = rank * (THREADS / 32) + warp; m < rows; m += ranks * (THREADS / 32)) {
        float4 v = cluster_sum(base + (m * BN + c) * 4, ranks);
        v = make_float4(v.x + b.x, v.y + b.y, v.z + b.z, v.w + b.w);
        if (p.act == H3B_ACT_GELU_TANH)
          v = make_float4(mxgemm::gelu_tanh_f32(v.x), mxgemm::gelu_tanh_f32(v.y),
                          mxgemm::gelu_tanh_f32(v.z), mxgemm::gelu_tanh_f32(v.w));
        if (residual) {
          const float4 r = load4(residual + (size_t)(m0 + m) * p.ldr + n);
          v = make_float4(v.x + r.x, v.y + r.y, v.z + r.z, v.w + r.w);
        }
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (size_t)(m0 + m) * p.ldd + n) =
            make_uint2(mx::pack2(v.x, v.y, T()), mx::pack2(v.z, v.w, T()));
      }
    }
  } else {
    // rows 0-63 of the weight tile are values, 64-127 their gates: 16 threads
    // cover a row's 64 hidden columns, eight of them one 32-value block
    const int c = (threadIdx.x & 15) * 4;
    const int F = p.N >> 1, f = (n0 >> 1) + c;
    const int pass = THREADS / 16;       // rows; all lanes of a warp stay in the loop
    for (int i = rank * pass; i < rows; i += ranks * pass) {
      const int m = i + (int)(threadIdx.x >> 4);
      float h[4] = {0.f, 0.f, 0.f, 0.f};
      if (m < rows) {
        const float4 v = cluster_sum(base + (m * BN + c) * 4, ranks);
        const float4 g = cluster_sum(base + (m * BN + 64 + c) * 4, ranks);
        h[0] = mxgemm::swiglu_f32(v.x, g.x);
        h[1] = mxgemm::swiglu_f32(v.y, g.y);
        h[2] = mxgemm::swiglu_f32(v.z, g.z);
        h[3] = mxgemm::swiglu_f32(v.w, g.w);
      }
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) bits = max(bits, __float_as_uint(h[i]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = 1; o < 8; o *= 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
      const uint32_t s = mx::scale_byte(bits);
      const float inv = mx::scale_inverse(s);
      const uint32_t code = f32x2_to_e2m1x2(h[0] * inv, h[1] * inv) |
                            f32x2_to_e2m1x2(h[2] * inv, h[3] * inv) << 8;
      if (m < rows) {
        *reinterpret_cast<uint16_t*>(p.q_out + (size_t)(m0 + m) * (F >> 1) + (f >> 1)) =
            (uint16_t)(inv != 0.f ? code : 0u);
        if (!(threadIdx.x & 7)) p.sf_out[sf_swizzled_offset(m0 + m, f >> 5, F >> 7)] = (uint8_t)s;
      }
    }
  }
  // nobody leaves while its partial is read; the loads above have returned, and
  // the results need not be out before the others may go
  if (ranks > 1) cluster_sync_relaxed();
}

}  // namespace mxrows
}  // namespace h3b
