// Windowed attention of a few new tokens per sequence against a cache, lengths
// read on the device (so a captured launch serves every step): the visibility
// rule of attention_window.cuh for queries at positions len - n_new ... len - 1.
//
// Bound by reading the visible keys and values once: 32 uneven sequences (503 MB)
// in 75.7 us, 6.6 TB/s; one sequence of 4100 keys (16.8 MB) in 7.6 us, where
// latencies are half of it.  The rows that share a key head, n_new tokens times
// the group's query heads, are the 8 (or twice 8) columns of mma.sync m16n8k16
// products with the keys on the other side: S^T = K Q^T and O^T = V^T P^T, which
// for up to 8 rows takes half the instructions of the form with 16 rows of
// queries.  A warp's work is one pass, with a running maximum and sum, over key
// tiles of 16, K and V copied by cp.async into its own ring of
// stages (no barrier among warps); all fragments of K, and of V, are asked for
// before the arithmetic that uses them.  A cluster of CTAs along the keys shares
// a (sequence, key head): tile i belongs to warp i mod (cluster warps), and the
// partial results (maximum, sum, unnormalised output, all fp32) are joined first
// in a CTA's shared memory, then across the cluster: every CTA sends each rank
// the share of the rows' elements which that rank adds up (st.async, counted on
// the receiver's mbarrier; a cluster barrier at this place cost about 2000
// cycles, and another one before the exit), always in the same order.
#pragma once

#include "attention_window.cuh"

namespace h3b {
namespace wdec {

constexpr int kWarps = 4;            // 96 KiB of rings (D = 128): two CTAs per SM
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;           // keys per tile
constexpr int kMaxCluster = 8;

// Rings of three stages: 96 KiB (D = 128), two CTAs per SM.  NT: 8-row columns
// of the products.
template <int D, int NT>
struct Smem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kStages = 3;
  static constexpr int TILE = kKeys * D * 2;                  // K or V of one stage
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WARP = kStages * STAGE;
  static constexpr int RING = kWarps * WARP;
  // after the pass: per warp the rows of D (+ 4, which spreads a warp's stores
  // over the banks) fp32 and their (max, sum)
  static constexpr int PITCH = D + 4;
  static constexpr int PART = kRows * PITCH * 4 + kRows * 8;
  // received from the cluster, per rank: its share's elements (float4s) and
  // every row's (max, sum)
  static constexpr int RECV = RING > kWarps * PART ? RING : kWarps * PART;
  static constexpr int BYTES = RECV + kRows * D * 4 + kMaxCluster * 16 + kMaxCluster * kRows * 8;
};

struct Args {
  const void *q, *k, *v;
  void* out;                        // [B, n_new, H, D] contiguous
  const int32_t* len;               // [B] keys in use, the new tokens' own included
  long long q_b, q_t, q_h;          // strides in elements
  long long k_b, k_s, k_h, v_b, v_s, v_h;
  int room, n_new, H, kv_heads, group;
  int left, right, sinks, causal;
  float scale_log2;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// Transpose of an 8 x 8 matrix of 16-bit values held two per lane.
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, "
                 "{%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Asynchronous stores to a CTA of the cluster (addresses from mapa_shared),
// their bytes counted on that CTA's mbarrier.
__device__ __forceinline__ void st_async_f4(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::
          "r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void st_async_f2(uint32_t addr, float2 v, uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::
          "r"(addr), "f"(v.x), "f"(v.y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Joins (m, l) pairs: the weight of a partial whose maximum is m in a total
// whose maximum is top; a partial that saw nothing (m = -inf) weighs 0.
__device__ __forceinline__ float weight(float m, float top) {
  return m == -INFINITY ? 0.f : attn::ex2(m - top);
}

template <int D, typename T, int NT>
__global__ void __launch_bounds__(kThreads) k_window_decode(const __grid_constant__ Args p) {
  using L = Smem<D, NT>;
  constexpr int kRows = L::kRows;
  constexpr int CH = D / 8;                       // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t recv_bar;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), ranks = (int)cluster_nctarank();
  const int rows_all = p.n_new * p.group;
  const int row_tiles = (rows_all + kRows - 1) / kRows;
  const int kvh = blockIdx.y / row_tiles;
  const int row0 = (blockIdx.y % row_tiles) * kRows;
  const int rows = min(kRows, rows_all - row0);
  const int b = blockIdx.z;
  // the cluster's receive barriers exist before anything is sent (waited for
  // after the pass)
  const int f4s = rows * (D / 4);                 // the result's float4s; rank r adds up
  const int share = (f4s + ranks - 1) / ranks;    // [r * share, (r + 1) * share)
  const int mine = max(0, min(share, f4s - rank * share));
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&recv_bar), 1);
    fence_mbar_init();
    mbar_expect_tx(smem_u32(&recv_bar), (uint32_t)(ranks * (mine * 16 + rows * 8)));
  }
  __syncthreads();
  cluster_arrive();
  grid_wait();
  grid_launch_dependents();
  const int n = min(max(p.len[b], 0), p.room);

  // keys that any of this tile's rows sees: [0, sink_end) and [lo, end), visited
  // as one list of `total` keys
  const int t0 = row0 / p.group, t1 = (row0 + rows - 1) / p.group;
  const int p0 = n - p.n_new + t0, p1 = n - p.n_new + t1;
  const int top = p.causal ? min(p1, n - 1) : n - 1;
  int sink_end = max(0, min(p.sinks, top + 1));
  int lo = max(0, p0 - p.left);
  int end = min(top, p1 + p.right) + 1;
  if (end > lo && sink_end >= lo) {               // they touch: one range from 0
    end = max(end, sink_end);
    lo = 0;
    sink_end = 0;
  }
  const int total = sink_end + max(0, end - lo);
  const int tiles = (total + kKeys - 1) / kKeys;

  // Q^T as B fragments: row lane / 4 of each 8, dims (lane % 4) * 2 + {0, 1} and + 8
  uint32_t qf[D / 16][NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = j * 8 + (lane >> 2);
    const bool ok = r < rows;
    const int t = (row0 + min(r, rows - 1)) / p.group;
    const int g = (row0 + min(r, rows - 1)) % p.group;
    const T* q = static_cast<const T*>(p.q) + b * p.q_b + t * p.q_t +
                 (long long)(kvh * p.group + g) * p.q_h + (lane & 3) * 2;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      qf[kk][j][0] = ok ? *reinterpret_cast<const uint32_t*>(q + kk * 16) : 0u;
      qf[kk][j][1] = ok ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8) : 0u;
    }
  }
  // this lane's rows in the products: j * 8 + (lane % 4) * 2 + {0, 1}
  int pos[NT][2];                                 // their key positions
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = min(j * 8 + (lane & 3) * 2 + h, rows - 1);
      pos[j][h] = n - p.n_new + (row0 + r) / p.group;
      m[j][h] = -INFINITY;
      l[j][h] = 0.f;
    }
  float o[D / 16][NT][4];                         // O^T: dims 16 d + lane / 4 and + 8
#pragma unroll
  for (int d = 0; d < D / 16; ++d)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[d][j][c] = 0.f;

  const T* kb = static_cast<const T*>(p.k) + b * p.k_b + kvh * p.k_h;
  const T* vb = static_cast<const T*>(p.v) + b * p.v_b + kvh * p.v_h;
  const uint32_t ring = smem_u32(smem) + warp * L::WARP;
  const int first = rank * kWarps + warp, stride = ranks * kWarps;

  // copy tile i into stage s: a lane's chunk of every 32 / CH-th row; a tile
  // inside one region advances one pointer per matrix, one that straddles the
  // sinks' end or the last key (zeros behind it) asks for each row
  const int ch0 = lane % CH, r0 = lane / CH;
  constexpr int RPP = 32 / CH;                    // rows per pass
  auto fetch = [&](int i, int s) {
    if (i < tiles) {
      const int u0 = i * kKeys;
      const uint32_t st = ring + s * L::STAGE;
      if (u0 + kKeys <= total && (u0 >= sink_end || u0 + kKeys <= sink_end)) {
        const long long key = (u0 < sink_end ? u0 : lo + (u0 - sink_end)) + r0;
        const T* kp = kb + key * p.k_s + ch0 * 8;
        const T* vp = vb + key * p.v_s + ch0 * 8;
#pragma unroll
        for (int r = 0; r < kKeys; r += RPP) {
          const uint32_t dst = st + (r + r0) * (D * 2) + ((ch0 ^ ((r + r0) & 7)) << 4);
          cp_async16(dst, kp, 16);
          cp_async16(dst + L::TILE, vp, 16);
          kp += RPP * p.k_s;
          vp += RPP * p.v_s;
        }
      } else {
#pragma unroll 1
        for (int r = r0; r < kKeys; r += RPP) {
          const int u = u0 + r;
          const bool ok = u < total;
          const long long key = !ok ? 0 : u < sink_end ? u : lo + (u - sink_end);
          const uint32_t dst = st + r * (D * 2) + ((ch0 ^ (r & 7)) << 4);
          cp_async16(dst, kb + key * p.k_s + ch0 * 8, ok ? 16 : 0);
          cp_async16(dst + L::TILE, vb + key * p.v_s + ch0 * 8, ok ? 16 : 0);
        }
      }
    }
    cp_commit();
  };
  // ldmatrix: lane i of the warp gives the address of row i % 8 of matrix i / 8
  const int lr = lane & 7, lm = lane >> 3;

#pragma unroll
  for (int s = 0; s < L::kStages - 1; ++s) fetch(first + s * stride, s);
  int s = 0;
  for (int i = first; i < tiles; i += stride) {
    cp_wait<L::kStages - 2>();
    __syncwarp();
    const uint32_t ks = ring + s * L::STAGE, vs = ks + L::TILE;
    uint32_t f[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      // K as A: keys 0-7 and 8-15 of dims 0-7, then of dims 8-15
      const int r = lr + (lm & 1) * 8, ch = kk * 2 + (lm >> 1);
      ldsm4(ks + r * (D * 2) + ((ch ^ (r & 7)) << 4), f[kk]);
    }
    // into the stage of the last tile, which every lane read before the
    // __syncwarp above
    fetch(i + (L::kStages - 1) * stride, (s + L::kStages - 1) % L::kStages);
    // S^T, even and odd k-steps apart: shorter chains of MMAs
    float sc[NT][4], sd[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) sc[j][c] = sd[j][c] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        mma16816<T>(kk & 1 ? sd[j] : sc[j], f[kk], qf[kk][j][0], qf[kk][j][1]);
    uint32_t g[D / 16][4];
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) {
      // V^T as A: dims 0-7 and 8-15 of keys 0-7, then of keys 8-15
      const int r = lr + (lm >> 1) * 8, ch = dd * 2 + (lm & 1);
      ldsm4_t(vs + r * (D * 2) + ((ch ^ (r & 7)) << 4), g[dd]);
    }
    // visibility and scaling (log2 units): this lane's keys lane / 4 and + 8
    const int u0 = i * kKeys + (lane >> 2);
    uint32_t pf[NT][2];
    float al[NT][2];
    bool moved = false;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int u = u0 + (c >> 1) * 8;
        const int key = u < sink_end ? u : lo + (u - sink_end);
        const int ps = pos[j][c & 1];
        const bool near = key >= ps - p.left && key <= ps + p.right;
        const bool seen = u < total && (near || key < p.sinks) && (!p.causal || key <= ps);
        sc[j][c] = seen ? (sc[j][c] + sd[j][c]) * p.scale_log2 : -INFINITY;
        mx[c & 1] = fmaxf(mx[c & 1], sc[j][c]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int x = 4; x < 32; x *= 2) mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], x));
        const float mn = fmaxf(m[j][h], mx[h]);
        const float mb = mn == -INFINITY ? 0.f : mn;
        al[j][h] = attn::ex2(m[j][h] - mb);       // 0 while nothing was seen
        m[j][h] = mn;
        moved |= al[j][h] != 1.f;
        sc[j][h] = attn::ex2(sc[j][h] - mb);
        sc[j][h + 2] = attn::ex2(sc[j][h + 2] - mb);
        l[j][h] = l[j][h] * al[j][h] + (sc[j][h] + sc[j][h + 2]);
      }
      // P^T as B: the 8 x 8 halves transposed
      pf[j][0] = movm(wattn::pack16<T>(sc[j][0], sc[j][1]));
      pf[j][1] = movm(wattn::pack16<T>(sc[j][2], sc[j][3]));
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[d][j][c] *= al[j][c & 1];
    }
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int j = 0; j < NT; ++j) mma16816<T>(o[dd][j], g[dd], pf[j][0], pf[j][1]);
    s = (s + 1) % L::kStages;
  }
  cp_wait<0>();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 4; x < 32; x *= 2) l[j][h] += __shfl_xor_sync(0xffffffffu, l[j][h], x);
  __syncthreads();                                // every warp is done with its ring

  // partials: part w at w * PART: O [rows][PITCH] fp32, then (m, l) per row
  auto part_o = [&](int w) { return reinterpret_cast<float*>(smem + w * L::PART); };
  auto part_ml = [&](int w) {
    return reinterpret_cast<float2*>(smem + w * L::PART + kRows * L::PITCH * 4);
  };
  {
    float* po = part_o(warp);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = j * 8 + (lane & 3) * 2 + h;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          po[r * L::PITCH + d * 16 + (lane >> 2)] = o[d][j][h];
          po[r * L::PITCH + d * 16 + (lane >> 2) + 8] = o[d][j][h + 2];
        }
        if (lane < 4) part_ml(warp)[r] = make_float2(m[j][h], l[j][h]);
      }
  }
  cluster_wait();                                 // the receivers are ready
  __syncthreads();
  // the CTA's own total: each warp's weight per row once, in the place of its
  // maximum; the row's (max, sum) goes to every rank
  const uint32_t recv = smem_u32(smem) + L::RECV, bar = smem_u32(&recv_bar);
  const uint32_t recv_ml = recv + share * ranks * 16;
  if (threadIdx.x < rows) {
    const int r = threadIdx.x;
    float2 ml[kWarps];
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      ml[w] = part_ml(w)[r];
      mm = fmaxf(mm, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = weight(ml[w].x, mm);
      ll += f * ml[w].y;
      part_ml(w)[r].x = f;
    }
    for (int c = 0; c < ranks; ++c)
      st_async_f2(mapa_shared(recv_ml + (rank * kRows + r) * 8, c), make_float2(mm, ll),
                  mapa_shared(bar, c));
  }
  __syncthreads();
  for (int e = threadIdx.x; e < f4s; e += kThreads) {
    const int r = e / (D / 4), c4 = e % (D / 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = part_ml(w)[r].x;
      const float4 v = *reinterpret_cast<const float4*>(part_o(w) + r * L::PITCH + c4 * 4);
      acc = make_float4(acc.x + f * v.x, acc.y + f * v.y, acc.z + f * v.z, acc.w + f * v.w);
    }
    const int to = e / share;
    st_async_f4(mapa_shared(recv + (rank * share + e - to * share) * 16, to), acc,
                mapa_shared(bar, to));
  }
  // the cluster's total of this rank's share, in rank order
  if (!mbar_wait(bar, 0, nullptr)) {
    record_error(H3B_ERR_TIMEOUT);
    return;
  }
  const float4* ro = reinterpret_cast<const float4*>(smem + L::RECV);
  const float2* rml = reinterpret_cast<const float2*>(smem + L::RECV + share * ranks * 16);
  for (int i = threadIdx.x; i < mine; i += kThreads) {
    const int e = rank * share + i, r = e / (D / 4), d = (e % (D / 4)) * 4;
    float mm = -INFINITY, ll = 0.f;
    for (int c = 0; c < ranks; ++c) mm = fmaxf(mm, rml[c * kRows + r].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < ranks; ++c) {
      const float f = weight(rml[c * kRows + r].x, mm);
      const float4 v = ro[c * share + i];
      ll += f * rml[c * kRows + r].y;
      acc = make_float4(acc.x + f * v.x, acc.y + f * v.y, acc.z + f * v.z, acc.w + f * v.w);
    }
    const int t = (row0 + r) / p.group, g = (row0 + r) % p.group;
    const size_t at = (((size_t)b * p.n_new + t) * p.H + kvh * p.group + g) * D + d;
    const float inv = 1.0f / ll;
    // does the row see any key at all (one that does, and only logits of -inf, is NaN)
    const int ps = n - p.n_new + t;
    const int top_r = p.causal ? min(ps, n - 1) : n - 1;
    const bool some = min(p.sinks, top_r + 1) > 0 || min(ps + p.right, top_r) >= max(0, ps - p.left);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at) =
        some ? make_uint2(wattn::pack16<T>(acc.x * inv, acc.y * inv),
                               wattn::pack16<T>(acc.z * inv, acc.w * inv))
                  : make_uint2(0u, 0u);
  }
}

}  // namespace wdec
}  // namespace h3b
