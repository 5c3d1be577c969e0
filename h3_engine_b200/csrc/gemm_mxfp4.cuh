// MXFP4 x MXFP4 GEMM on the 5th-generation tensor cores (sm_100a):
//   D[m, n] = sum_k A[m, k] 2^ea[m, k/32]  B[n, k] 2^eb[n, k/32]
// E2M1 codes, one E8M0 scale per 32 values of K, fp32 accumulation
// (tcgen05.mma kind::mxf4, scale_vec::2X: K = 64 and two scales per row and
// instruction).
//
// The scales are half as many as NVFP4's: one 128 x 4 tile of them (512 bytes,
// one tcgen05.cp of 4 TMEM columns) serves two MMA k-steps, chosen by the
// scale-factor id of the instruction descriptor (bytes 0-1 or 2-3 of each 32-bit
// column).  K is any multiple of 32: TMA fills the codes past K with zeros, the
// last k-block issues only the k-steps that hold values, and the scale bytes
// past K/32 are zeros (2^-127) by the format.
//
// Bound by the tensor core's pipe: 256 values of K of a 256 x 256 tile take about
// 650 clocks, 512 of them the MMAs and the rest the copies of the scales, which
// share the pipe.  13383 x 28672 x 5376: 735 us, 5.6 PFLOP/s.
#pragma once

#include "common.cuh"
#include "gemm_nvfp4.cuh"
#include "quant_mx.cuh"

namespace h3b {
namespace mxgemm {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int KB_ELEMS = 256;                 // values of K per pipeline stage
constexpr int KB_BYTES = KB_ELEMS / 2;
constexpr int SF_ATOM = 512;                  // scales of 128 rows x 128 values
constexpr int KB_ATOMS = KB_ELEMS / 128;
constexpr int EPI_WARPS = 8;
constexpr int OUT_BOX_BYTES = 4096;           // 32 rows x 128 bytes, one 128B-swizzled box
constexpr int OUT_WARP_BYTES = 2 * OUT_BOX_BYTES;   // both halves of a warp's 128 columns
constexpr int OUT_COLS = 64;                  // 16-bit columns per TMA store
constexpr int THREADS = 64 + EPI_WARPS * 32;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t ACC_COL = 0;
constexpr uint32_t SF_COL = 256;
constexpr uint32_t SF_STAGE_COLS = KB_ATOMS * 4 + KB_ATOMS * 8;

// Instruction descriptor: A and B E2M1 (bits 7, 10), UE8M0 scales (bit 23),
// N >> 3 at 17, M >> 7 at 27; scale-factor ids of B at 4 and of A at 29
// (0 or 2: which half of a 32-bit scale column).
__host__ __device__ constexpr uint32_t idesc(uint32_t m, uint32_t n, uint32_t id) {
  return (id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) |
         (id << 29);
}

// Arrive on an mbarrier of a CTA of the cluster without ordering earlier memory
// operations (the arrival itself is all that the waiter needs).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t remote_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar)
               : "memory");
}

enum Epilogue { kOut = 0, kSwigluQuant = 1, kOutGelu = 2 };

struct Args {
  CUtensorMap tmap_a;      // u8 [M, K/2], box 128 B x 128 rows, 128B swizzle
  CUtensorMap tmap_b;      // u8 [N, K/2], box 128 B x 128 rows, 128B swizzle
  CUtensorMap tmap_d;      // kOut(Gelu): 16-bit [M, N] (pitch ldd), box 64 x 32, 128B swizzle
  const uint8_t* sfa;      // blocked scales, M padded to 128 rows
  const uint8_t* sfb;
  const void* bias;        // [N], type of D
  CUtensorMap tmap_r;      // the residual (pitch ldr), as tmap_d
  int residual;            // there is one
  uint8_t* q_out;          // kSwigluQuant: codes u8 [M, N/4]
  uint8_t* sf_out;         // and their blocked scales
  int M, N, K;
  int sf_tiles_k;          // 512-byte scale tiles per 128-row block
  int n_tiles;
  int early;               // the next launch may come up under this one
};

__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) { return bf16x2_to_f2(w); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// GELU (tanh form) as v * sigmoid(2 u), u = sqrt(2 / pi) (v + 0.044715 v^3):
// (1 + tanh u) / 2 is sigmoid(2 u), so nothing cancels, and the exponential's
// relative error (2 + 1.2 |2 u| steps of 2^-23) is all there is.
__device__ __forceinline__ float gelu_tanh_f32(float v) {
  const float u2 = 1.5957691216057308f * fmaf(0.044715f * v, v * v, v);
  return __fdividef(v, 1.0f + __expf(-u2));
}

// The residual of a warp's 32 rows x 128 columns into its staging boxes, under
// the MMAs of the tile; false where the warp has none.
__device__ __forceinline__ bool residual_load(const Args& p, int m0, int n0, int half, int qd,
                                              int lane, uint32_t stage_s, uint32_t bar) {
  const int n_base = n0 + half * 128, row = m0 + qd * 32;
  if (!p.residual || n_base >= p.N || row >= p.M) return false;
  if (lane == 0) {
    bulk_wait_read0();                                // the last tile's boxes have been read
    const int boxes = n_base + OUT_COLS < p.N ? 2 : 1;
    mbar_expect_tx(bar, (uint32_t)boxes * OUT_BOX_BYTES);
    for (int c = 0; c < boxes; ++c)
      tma_load_2d(stage_s + c * OUT_BOX_BYTES, &p.tmap_r, n_base + c * OUT_COLS, row, bar);
  }
  __syncwarp();
  return true;
}

// Epilogue of one warp's 32 rows x 128 accumulator columns: columns
// n0 + 128 * half .. of a tile whose rows start at m0.  With a residual the
// boxes hold it, and each 16 bytes are replaced by the result (13383 x 5376 x
// 7168: 200 us, 204 with the residual read from global memory here, a row per
// lane; K = 2048: 84 and 146, 1025 x 2016 x 5504: 14.1 and 17.8).
template <typename T, bool GELU>
__device__ __forceinline__ void epilogue_out(const Args& p, const uint32_t (&acc)[128], int m0,
                                             int n0, int half, int qd, int lane, uint8_t* stage,
                                             uint32_t stage_s) {
  const int n_base = n0 + half * 128;
  if (n_base >= p.N || m0 + qd * 32 >= p.M) return;   // warp-uniform
  const T* bias = static_cast<const T*>(p.bias);
  if (!p.residual) {
    if (lane == 0) bulk_wait_read0();                 // the last tile's boxes have been read
    __syncwarp();
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (n_base + c * OUT_COLS >= p.N) break;          // the box would start past N
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = n_base + c * OUT_COLS + j * 8;
      const bool col_ok = col < p.N;                  // N % 8 == 0: all 8 or none
      float2 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = make_float2(__uint_as_float(acc[c * 64 + j * 8 + 2 * e]),
                           __uint_as_float(acc[c * 64 + j * 8 + 2 * e + 1]));
      if (bias && col_ok) {
        const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias + col));
        const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = add2(v[e], unpack2(bw[e], T()));
      }
      if (GELU) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = make_float2(gelu_tanh_f32(v[e].x), gelu_tanh_f32(v[e].y));
      }
      // 128B swizzle: 16-byte chunk j of row `lane` sits at chunk j ^ (lane % 8)
      uint4* const at = reinterpret_cast<uint4*>(stage + c * OUT_BOX_BYTES + lane * 128 +
                                                 ((j ^ (lane & 7)) << 4));
      if (p.residual) {
        const uint4 b = *at;
        const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = add2(v[e], unpack2(bw[e], T()));
      }
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = mx::pack2(v[e].x, v[e].y, T());
      *at = make_uint4(o[0], o[1], o[2], o[3]);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(&p.tmap_d, stage_s + c * OUT_BOX_BYTES, n_base + c * OUT_COLS, m0 + qd * 32);
      bulk_commit();
    }
  }
}

// h = v * silu(g), in fp32 all the way to the E2M1 rounding.  __expf's
// relative error (2^-21 near zero, growing with |g|) moves a code only where h
// sits that close to a rounding boundary.
__device__ __forceinline__ float swiglu_f32(float v, float g) {
  return v * __fdividef(g, 1.0f + __expf(-g));
}

// SwiGLU epilogue that writes the hidden activation as MXFP4: the 128
// accumulator columns are 64 values and their 64 gates, so a lane holds two
// whole 32-value blocks of its row; block maximum, scale and codes need no
// other lane, and the hidden activation never exists in 16 bits.
__device__ __forceinline__ void epilogue_swiglu_quant(const Args& p, const uint32_t (&acc)[128],
                                                      int m0, int n0, int half, int qd, int lane) {
  const int row = m0 + qd * 32 + lane;
  if (row >= p.M) return;
  const int f0 = (n0 >> 1) + half * 64;               // first hidden column
  const int64_t F = p.N >> 1;
  uint32_t s[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    float h[32];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      h[i] = swiglu_f32(__uint_as_float(acc[b * 32 + i]), __uint_as_float(acc[64 + b * 32 + i]));
      m = max(m, __float_as_uint(h[i]) & 0x7FFFFFFFu);
    }
    s[b] = mx::scale_byte(m);
    const float inv = mx::scale_inverse(s[b]);
    uint32_t o[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = h[w * 8 + i];
      o[w] = mx::codes8(v, inv);
    }
    *reinterpret_cast<uint4*>(p.q_out + (size_t)row * (F >> 1) + (f0 >> 1) + b * 16) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
  // F % 128 == 0: no padding columns, and the pair never straddles a tile
  *reinterpret_cast<uint16_t*>(p.sf_out + sf_swizzled_offset(row, f0 >> 5, F >> 7)) =
      (uint16_t)(s[0] | (s[1] << 8));
}

// ============================================================================
// CTA-pair kernel (cluster of 2): one 256 x 256 tile per pair, the MMA in its
// cta_group::2 form.  CTA r loads rows m0 + 128 r .. of A with their scales,
// rows n0 + 128 r .. of B (its half of the tile's N) and the scales of all 256
// B rows; every load counts its bytes on the leader's full barrier
// (cta_group::2 form, no multicast).  The leader's MMA warp alone issues, for
// both SMs: per 128 values of K three scale copies and two MMAs.  Scale tiles
// come through tensor maps so that rows and columns outside the operand read
// as zeros.  Protocol, bounds and teardown as in the NVFP4 pair kernel.
// ============================================================================
//
// Between tiles the tensor core waits for the accumulator: commit, the epilogue
// warps' tcgen05.ld (about 100 cycles), their arrival on the leader's barrier.
// That arrival is a relaxed one (nothing but registers was produced before it):
// a release at cluster scope made it wait for the warp's earlier stores, 1900
// cycles of the 21000 that a tile with K = 7168 took.
constexpr int P_STAGES = 4;
constexpr int P_A_BYTES = 128 * KB_BYTES;
constexpr int P_B_BYTES = 128 * KB_BYTES;
constexpr int P_SFA_BYTES = KB_ATOMS * SF_ATOM;
constexpr int P_SFB_BYTES = 2 * KB_ATOMS * SF_ATOM;
constexpr int P_STAGE_BYTES = P_A_BYTES + P_B_BYTES + P_SFA_BYTES + P_SFB_BYTES;
constexpr int P_OUT_OFFSET = P_STAGES * P_STAGE_BYTES;
constexpr int P_BAR_OFFSET = P_OUT_OFFSET + EPI_WARPS * OUT_WARP_BYTES;
constexpr int P_SMEM_BYTES = P_BAR_OFFSET + 256 + 1024;
static_assert(P_STAGE_BYTES % 1024 == 0 && P_OUT_OFFSET % 1024 == 0, "swizzle alignment");
static_assert(SF_COL + P_STAGES * SF_STAGE_COLS <= TMEM_COLS, "TMEM budget");
static_assert(P_SMEM_BYTES <= 232448, "shared memory budget");

struct PairArgs {
  Args base;
  CUtensorMap tmap_sfa;    // u64 [128-row blocks, scale tiles * 64], box 128 x 1 (one k-block)
  CUtensorMap tmap_sfb;    // the same for B, box 128 x 2
  int m_tiles;             // 256-row tiles
  int group;               // tile rows per raster group
};

// Tile t of the raster: groups of `group` tile rows, column by column inside a
// group, so that the tiles running at one time share A rows and B columns.
__device__ __forceinline__ void pair_tile(const PairArgs& p, int t, int& m, int& n) {
  const int per = p.group * p.base.n_tiles;
  const int g = t / per, r = t - g * per;
  const int rows = min(p.group, p.m_tiles - g * p.group);
  n = r / rows;
  m = g * p.group + (r - n * rows);
}

__device__ __forceinline__ void kpair_pair_elect(uint32_t sfa_t, uint64_t sfa_d, uint32_t sfb_t,
                                                 uint64_t sfb_d0, uint64_t sfb_d1, uint32_t d_tmem,
                                                 uint64_t a_desc, uint64_t b_desc,
                                                 uint32_t accumulate, uint32_t second) {
  asm volatile(
      "{\n\t.reg .pred p, e, f;\n\t"
      "setp.ne.b32 p, %9, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%2], %3;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%4], %5;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X"
      " [%6], %7, %8, %10, [%0], [%2], p;\n\t"
      "setp.ne.and.b32 f, %12, 0, e;\n\t"
      "setp.eq.u32 p, 0, 0;\n\t"
      "@f tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X"
      " [%6], %13, %14, %11, [%0], [%2], p;\n\t}" ::"r"(sfa_t),
      "l"(sfa_d), "r"(sfb_t), "l"(sfb_d0), "r"(sfb_t + 4), "l"(sfb_d1), "r"(d_tmem), "l"(a_desc),
      "l"(b_desc), "r"(accumulate), "r"(idesc(256, 256, 0)), "r"(idesc(256, 256, 2)),
      "r"(second), "l"(a_desc + 2), "l"(b_desc + 2)
      : "memory");
}

template <typename T, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    k_gemm_mxfp4_pair(const __grid_constant__ PairArgs pa) {
  const Args& p = pa.base;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P_BAR_OFFSET);
  uint64_t* full = bars;                       // leader: both CTAs' loads of a stage
  uint64_t* empty = bars + P_STAGES;           // both: stage consumed (leader's commit)
  uint64_t* acc_full = bars + 2 * P_STAGES;    // both: accumulator ready
  uint64_t* acc_empty = bars + 2 * P_STAGES + 1;   // leader: both CTAs drained it
  uint64_t* drain = bars + 2 * P_STAGES + 2;
  uint64_t* bye = bars + 2 * P_STAGES + 3;     // both: the peer is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * P_STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint64_t* res_full = bars + 16;              // per epilogue warp: the residual's boxes

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int num_kb = (p.K + KB_ELEMS - 1) / KB_ELEMS;
  const int pair_id = (int)(blockIdx.x >> 1);
  const int num_pairs = (int)(gridDim.x >> 1);
  const int num_tiles = pa.m_tiles * p.n_tiles;

  auto sA = [&](int s) { return smem + s * P_STAGE_BYTES; };
  auto sB = [&](int s) { return smem + s * P_STAGE_BYTES + P_A_BYTES; };
  auto sSFA = [&](int s) { return smem + s * P_STAGE_BYTES + P_A_BYTES + P_B_BYTES; };
  auto sSFB = [&](int s) {
    return smem + s * P_STAGE_BYTES + P_A_BYTES + P_B_BYTES + P_SFA_BYTES;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < P_STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(acc_full), 1);
    mbar_init(smem_u32(acc_empty), 2 * EPI_WARPS);
    mbar_init(smem_u32(drain), 1);
    mbar_init(smem_u32(bye), 1);
    for (int i = 0; i < EPI_WARPS; ++i) mbar_init(smem_u32(&res_full[i]), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  // both CTAs' barriers exist before any load or arrival reaches them
  cluster_sync_all();
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
      prefetch_tmap(&p.tmap_a);
      prefetch_tmap(&p.tmap_b);
      prefetch_tmap(&pa.tmap_sfa);
      prefetch_tmap(&pa.tmap_sfb);
      auto load_b = [&](int s, int kb, int n0) {
        const uint32_t lb = mapa_shared(smem_u32(&full[s]), 0);
        if (rank == 0) mbar_expect_tx(smem_u32(&full[s]), 2 * P_STAGE_BYTES);
        tma_load_2d_pair(smem_u32(sB(s)), &p.tmap_b, kb * KB_BYTES, n0 + 128 * (int)rank, lb);
        tma_load_2d_pair(smem_u32(sSFB(s)), &pa.tmap_sfb, kb * KB_ATOMS * 64, n0 / 128, lb);
      };
      auto load_a = [&](int s, int kb, int m0) {
        const uint32_t lb = mapa_shared(smem_u32(&full[s]), 0);
        tma_load_2d_pair(smem_u32(sA(s)), &p.tmap_a, kb * KB_BYTES, m0 + 128 * (int)rank, lb);
        tma_load_2d_pair(smem_u32(sSFA(s)), &pa.tmap_sfa, kb * KB_ATOMS * 64,
                         m0 / 128 + (int)rank, lb);
      };
      uint32_t g = 0;
      bool ok = true;
      for (int t = pair_id; t < num_tiles && ok; t += num_pairs) {
        int mt, nt;
        pair_tile(pa, t, mt, nt);
        const int m0 = mt * 256, n0 = nt * BN;
        int kb = 0;
        if (t == pair_id) {
          // the weight's side of the ring fills before the chain's earlier
          // launch, which produces A, is done
          kb = min(num_kb, P_STAGES);
          for (int i = 0; i < kb; ++i) load_b(i, i, n0);
          grid_wait();
          for (int i = 0; i < kb; ++i) load_a(i, i, m0);
          g = kb;
        }
        for (; kb < num_kb; ++kb, ++g) {
          const int s = g % P_STAGES;
          const uint32_t ph = (g / P_STAGES) & 1;
          if (g >= P_STAGES && !mbar_wait(smem_u32(&empty[s]), ph ^ 1, abort_flag)) {
            fail();
            ok = false;
            break;
          }
          load_b(s, kb, n0);
          load_a(s, kb, m0);
        }
      }
      // tail: the release of every stage this CTA filled has arrived (the
      // leader's last commits reach this CTA's barriers before it can exit)
      for (uint32_t q = g > (uint32_t)P_STAGES ? g - P_STAGES : 0; q < g && ok; ++q) {
        if (!mbar_wait(smem_u32(&empty[q % P_STAGES]), (q / P_STAGES) & 1, abort_flag)) {
          fail();
          ok = false;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort_flag));
      };
      const int last_steps = (p.K - (num_kb - 1) * KB_ELEMS + 63) >> 6;
      uint32_t g = 0, i = 0;
      bool ok = true;
      for (int t = pair_id; t < num_tiles && ok; t += num_pairs, ++i) {
        if (i > 0 && !wait(acc_empty, (i - 1) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < num_kb; ++kb, ++g) {
          const int s = g % P_STAGES;
          const uint32_t ph = (g / P_STAGES) & 1;
          if (!wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int steps = kb == num_kb - 1 ? last_steps : 4;
          const uint32_t sf_t = tmem + SF_COL + s * SF_STAGE_COLS;
          const uint64_t sfa_d = desc_sf_atom(smem_u32(sSFA(s)));
          const uint64_t sfb_d = desc_sf_atom(smem_u32(sSFB(s)));
          const uint64_t a_d = desc_kmajor_sw128(smem_u32(sA(s)));
          const uint64_t b_d = desc_kmajor_sw128(smem_u32(sB(s)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h * 2 < steps)
              kpair_pair_elect(sf_t + h * 4, sfa_d + ((h * SF_ATOM) >> 4), sf_t + 8 + h * 8,
                               sfb_d + ((h * SF_ATOM) >> 4),
                               sfb_d + (((KB_ATOMS + h) * SF_ATOM) >> 4), tmem + ACC_COL,
                               a_d + h * 4, b_d + h * 4, (kb | h) != 0, h * 2 + 1 < steps);
          }
          tc_commit_pair_elect(smem_u32(&empty[s]), 0x3);
        }
        if (!ok) break;
        tc_commit_pair_elect(smem_u32(acc_full), 0x3);
      }
      if (!ok) {
        if (lane == 0) fail();
        tc_commit_pair_elect(smem_u32(drain), 0x1);
        mbar_wait(smem_u32(drain), 0, nullptr);
      }
    }
  } else {
    const int ew = warp - 2;
    const int qd = warp & 3;
    const int half = ew >> 2;
    uint8_t* stage = smem + P_OUT_OFFSET + ew * OUT_WARP_BYTES;
    const uint32_t stage_s = smem_u32(stage);
    const uint32_t leader_acc_empty = mapa_shared(smem_u32(acc_empty), 0);
    const uint32_t rbar = smem_u32(&res_full[ew]);
    uint32_t i = 0, loads = 0;
    grid_wait();                     // residual and D follow the chain's earlier launches
    if (p.early) grid_launch_dependents();
    if (EPI != kSwigluQuant && lane == 0) {
      prefetch_tmap(&p.tmap_d);
      if (p.residual) prefetch_tmap(&p.tmap_r);
    }
    for (int t = pair_id; t < num_tiles; t += num_pairs, ++i) {
      int mt, nt;
      pair_tile(pa, t, mt, nt);
      const int m0 = mt * 256 + 128 * (int)rank, n0 = nt * BN;
      const bool res = EPI != kSwigluQuant &&
                       residual_load(p, m0, n0, half, qd, lane, stage_s, rbar);
      bool ready = __all_sync(0xffffffffu, mbar_wait(smem_u32(acc_full), i & 1, abort_flag));
      // (bounded, but not cut short: no copy may still be landing at the exit)
      if (res) ready = __all_sync(0xffffffffu, mbar_wait(rbar, loads++ & 1, nullptr)) && ready;
      if (!ready) {
        fail();
        break;
      }
      tc_fence_after();
      uint32_t acc[128];
      const uint32_t taddr = tmem + ACC_COL + ((uint32_t)(qd * 32) << 16) + half * 128;
      tmem_ld_32x32b_x64(taddr, acc);
      tmem_ld_32x32b_x64(taddr + 64, acc + 64);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(leader_acc_empty);
      if (EPI == kSwigluQuant)
        epilogue_swiglu_quant(p, acc, m0, n0, half, qd, lane);
      else
        epilogue_out<T, EPI == kOutGelu>(p, acc, m0, n0, half, qd, lane, stage, stage_s);
    }
    if (EPI != kSwigluQuant && lane == 0) bulk_wait_read0();     // shared memory may go
  }

  tc_fence_before();
  __syncthreads();
  // the pair meets before either frees tensor memory or exits: the peer's
  // accumulator is written by the leader's MMAs, its loads count on the
  // leader's barriers
  if (threadIdx.x == 0) {
    mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(bye), rank ^ 1u));
    if (!mbar_wait(smem_u32(bye), 0, nullptr)) record_error(H3B_ERR_TIMEOUT);
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

}  // namespace mxgemm
}  // namespace h3b
