// Packed attention with a sliding window and sinks on the 5th-generation
// tensor cores: bf16 or fp16, head_dim 64 or 128, key heads shared by groups
// of query heads, fp32 softmax and accumulation.
//
// Query i of a document with n_q queries and n_k keys stands at key position
// p = i + n_k - n_q and sees key j iff
//     (p - left <= j <= p + right  or  j < sinks)  and  (not causal or j <= p).
// A query that sees no key gets zeros.
//
// One CTA = an item: two 128-row query tiles (A, B), or tile A alone, of one
// head of one document, in the roles and MMA order of attention.cuh.  Of the
// document's keys it visits only those that some query of the item sees: the
// sink keys [0, sink_end) and the window [lo, hi], each in steps of 128 or 64
// keys that start at 0 and at lo (TMA rows need no alignment, so the first step
// of the window starts at its first key); the two are one range where they
// touch.  A step that no query of tile A (or B) sees is skipped for that tile:
// neither its MMAs nor its softmax run, which is what the window's triangular
// ends cost least with.  Within a step a row's keys are words of 32, of
// which only those that some row of the warp does not see whole are masked.
//
// The grid is a number of full waves of items, one or two CTAs per SM, and a
// last partial wave whose items are split along their keys so that it fills
// the SMs too: the parts leave their unnormalised O, row maximum and sum (fp32) in a
// workspace, and the part that finishes last adds them up, in part order, so
// the result does not depend on which one that is.
//
// What bounds it: a tile's own cycle, softmax (1920 clocks per 128 x 128 step, of
// which the exponentials take at least 1024), P V (512) and Q K^T (512), which P
// over S makes take turns; the other tile's products run under the softmax.  8
// heads of 16384 rows that see 3200 keys each: 212 us, 962 TFLOP/s.  Measured and
// not taken: two S buffers per tile with steps of 64 keys (252 us: a product of
// 64 keys is bound by reading shared memory), two warpgroups per tile (232), a
// polynomial for part of the exponentials (222).
//
// Rows of V behind the last visible key of a step (the document's end, the
// next document, the gap behind the sinks) are cleared in shared memory before
// the MMA reads them: their P is 0, and 0 times what lies there must be 0.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"

namespace h3b {
namespace wattn {

constexpr int BQ = 128;
constexpr int MAX_DOCS = 64;          // documents per launch
constexpr int kPrefetchTiles = 4;

// Steps of 128 keys: all of tensor memory, one CTA per SM whose softmax
// warpgroups get the registers that the control warps give back.  With head_dim
// 64 the products are half as long while the softmax is not, and two softmax
// warps per scheduler leave it idle half the time; steps of 64 keys need half
// the registers and tensor memory, so two CTAs share an SM, where there are
// more CTAs than SMs (148 of them: 18.4 us in steps of 128, 20.5 in steps of
// 64; 240: 35.8 and 27.9).
template <int D, int KEYS>
struct Cfg {
  static constexpr int BK = KEYS;                          // keys per step
  static constexpr int CTAS = BK == 128 ? 1 : 2;           // per SM
  static constexpr int THREADS = BK == 128 ? 384 : 320;
  // P reaches the MMA in two pieces: the first 96 keys' products run under the
  // exponentials of the last 32 (in halves of 64 the second half's were waited
  // for: 16384 rows, 8 heads 218 us, 214 so)
  static constexpr int HALVES = BK / 64;
  static constexpr int P_FIRST = BK == 128 ? 96 : BK;
  static constexpr uint32_t TMEM_COLS = 512 / CTAS;
  static constexpr int Q_BOX = 128 * 128;                  // 128 rows x 64 columns
  static constexpr int Q_BYTES = (D / 64) * Q_BOX;
  static constexpr int KV_BOX = BK * 128;
  static constexpr int KV_BYTES = (D / 64) * KV_BOX;
  static constexpr int K_OFF = 2 * Q_BYTES;
  static constexpr int V_OFF = K_OFF + 2 * KV_BYTES;
  static constexpr int BAR_OFF = V_OFF + 2 * KV_BYTES;
  static constexpr int BYTES = BAR_OFF + 256 + 1024;
  static __device__ constexpr uint32_t s_col(int t) { return (uint32_t)(t * BK); }   // P over S
  static __device__ constexpr uint32_t o_col(int t) { return (uint32_t)(2 * BK + t * D); }
};
constexpr int kLaunchRegs = 168, kCtrlRegs = 72, kSoftmaxRegs = 216;
static_assert(128 * kCtrlRegs + 256 * kSoftmaxRegs <= Cfg<128, 128>::THREADS * kLaunchRegs,
              "register split");

struct Args {
  CUtensorMap tmap_q, tmap_k, tmap_v;      // 16-bit [rows, heads * D], 64 columns, 128B swizzle
  void* out;                               // [q rows, ldo]; head h at columns h * D
  long long ldo;
  int H, group;                            // query heads; query heads per key head
  float scale_log2;                        // softmax scale * log2(e)
  int left, right, sinks, causal;          // left, right < 2^30
  int item_rows;                           // queries per item: 256, or 128 (tile A only)
  int whole, parts;                        // items [0, whole) are whole, the others in parts,
                                           // each with places for `parts` of them
  float* partial;                          // [split item][part]: O [D/4][256][4], then (m, l) [256]
  int* done;                               // [split item]: parts finished (0 between launches)
  int ndocs;
  int q_start[MAX_DOCS], q_len[MAX_DOCS];
  int k_start[MAX_DOCS], k_len[MAX_DOCS];
  int item_end[MAX_DOCS];                  // cumulative item counts
  int parts_of[MAX_DOCS];                  // of a split item of the document, at most `parts`
};

// What queries at positions [p0, p1] of a document of n_k keys see: sink keys
// [0, sink_end) and the window [lo, hi] (empty when hi < lo).
struct Range {
  int sink_end, lo, hi;
  __device__ __forceinline__ Range(const Args& p, int n_k, int p0, int p1) {
    const int top = p.causal ? min(p1, n_k - 1) : n_k - 1;
    sink_end = max(0, min(p.sinks, top + 1));
    lo = max(0, p0 - p.left);
    hi = min(top, p1 + p.right);
  }
};

// The key steps of a CTA.
template <int BK>
struct Steps {
  int n_sink, n, lo, end, sink_end;        // window steps start at lo, end one past the last key
  int first = 0;                           // of this CTA's part; n counts its own
  __device__ __forceinline__ explicit Steps(const Range& r) {
    sink_end = r.sink_end;
    lo = r.lo;
    end = r.hi + 1;
    const int ns = (sink_end + BK - 1) / BK;
    const int nw = end > lo ? (end - lo + BK - 1) / BK : 0;
    n_sink = ns;
    n = ns + nw;
    if (nw > 0 && sink_end >= lo) {                     // they touch: one range
      n_sink = 0;
      lo = 0;
      end = max(end, sink_end);
      n = (end + BK - 1) / BK;
    }
  }
  __device__ __forceinline__ void take(int part, int parts) {
    first = (int)((long long)n * part / parts);
    n = (int)((long long)n * (part + 1) / parts) - first;
  }
  __device__ __forceinline__ int base(int j) const {
    j += first;
    return j < n_sink ? j * BK : lo + (j - n_sink) * BK;
  }
  __device__ __forceinline__ int valid(int j) const {
    return min(BK, (j + first < n_sink ? sink_end : end) - base(j));
  }
  // does a tile that sees `r` see any key of step j
  __device__ __forceinline__ bool needed(const Range& r, int j) const {
    const int b = base(j), e = b + valid(j);
    return b < r.sink_end || (b <= r.hi && e > r.lo && r.hi >= r.lo);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

// Warp-collective load and store of 16 consecutive 32-bit TMEM columns per lane.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// P = 2^(S * scale - m) of keys [K0, K0 + N) of a row, stored as 16-bit pairs over
// tensor memory from p_addr; adds them to acc.  P is rounded to 16 bits because
// the tensor core reads it so; the sum is of the unrounded fp32 values.  A masked
// key's S is -inf and its P 0.
template <typename T, int K0, int N, int BK>
__device__ __forceinline__ void softmax_store(const uint32_t (&sv)[BK], float scale_log2, float m,
                                              uint32_t p_addr, float2 (&acc)[2]) {
  const float2 sc = make_float2(scale_log2, scale_log2);
  const float2 nm = make_float2(-m, -m);
#pragma unroll
  for (int g = 0; g < N / 32; ++g) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const int k = K0 + g * 32 + 2 * c;
      const float2 x = fma2(make_float2(__uint_as_float(sv[k]), __uint_as_float(sv[k + 1])), sc, nm);
      const float2 e = make_float2(attn::ex2(x.x), attn::ex2(x.y));
      acc[c & 1] = add2(acc[c & 1], e);
      pk[c] = pack16<T>(e.x, e.y);
    }
    tmem_st_x16(p_addr + K0 / 2 + g * 16, pk);
  }
}

// Bits [a, b] of 32-bit word w of a 128-bit mask (a, b any ints).
__device__ __forceinline__ uint32_t span_word(int a, int b, int w) {
  const int lo = max(a - 32 * w, 0), hi = min(b - 32 * w, 31);
  if (hi < lo) return 0u;
  return (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
}

template <int D, int BK, typename T>
__global__ void __launch_bounds__(Cfg<D, BK>::THREADS, Cfg<D, BK>::CTAS)
    k_window_attn(const __grid_constant__ Args p) {
  using L = Cfg<D, BK>;
  // kind::f16: D fp32 (bit 4), A and B bf16 (bits 7, 10) or fp16 (0)
  constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
  constexpr uint32_t IDESC_QK =
      (1u << 4) | kType | ((uint32_t)(BK >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
  // P V: B = V is MN-major (head dim contiguous): bit 16
  constexpr uint32_t IDESC_PV =
      (1u << 4) | kType | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  // kv_full[j % 2]: V(j) and K(j + 1); kv_empty[j % 2]: after step j's last
  // MMAs, frees V stage j % 2 and K stage (j + 1) % 2 (K(0)'s release counts
  // as j = -1).  s_full / p_half / p_full count a tile's needed steps only.
  uint64_t* q_full = bars;           // 1
  uint64_t* kv_full = bars + 1;      // 2
  uint64_t* kv_empty = bars + 3;     // 2
  uint64_t* s_full = bars + 5;       // 2 (tile A, B)
  uint64_t* p_full = bars + 7;       // 2
  uint64_t* pv_done = bars + 9;      // 2: the last PV of a tile
  uint64_t* drain = bars + 11;       // 1
  uint64_t* p_half = bars + 12;      // 2: P of the first 96 keys of 128
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // work item (document, query-tile pair, head) and the part of its keys
  const int split = max(0, (int)blockIdx.x - p.whole) / p.parts;     // index of a split item
  const bool whole = (int)blockIdx.x < p.whole;
  const int part = whole ? 0 : ((int)blockIdx.x - p.whole) % p.parts;
  const int idx = whole ? (int)blockIdx.x : p.whole + split;
  int doc = 0;
  while (doc + 1 < p.ndocs && idx >= p.item_end[doc]) ++doc;
  const int item = idx - (doc > 0 ? p.item_end[doc - 1] : 0);
  const int parts = p.parts_of[doc];                      // of this item, where it is split
  if (!whole && part >= parts) return;                    // (part 0 of every item stays)
  const int n_q = p.q_len[doc], n_k = p.k_len[doc];
  const int pairs = (n_q + p.item_rows - 1) / p.item_rows;
  const int head = item / pairs;
  const int q0 = (item - head * pairs) * p.item_rows;     // first query in the document
  const int q_row = p.q_start[doc] + q0;
  const int k_row = p.k_start[doc];
  const int pos0 = q0 + n_k - n_q;                        // position of tile A's first row
  const int rows = min(p.item_rows, n_q - q0);            // queries of this item
  Steps<BK> st(Range(p, n_k, pos0, pos0 + rows - 1));
  if (!whole) st.take(part, parts);
  // what each tile sees; a tile without queries sees nothing
  auto tile_range = [&](int t) {
    const int n = min(BQ, rows - t * BQ);
    Range r(p, n_k, pos0 + t * BQ, pos0 + t * BQ + n - 1);
    if (n <= 0) {
      r.sink_end = 0;
      r.hi = -1;
      r.lo = 0;
    }
    return r;
  };

  const int qx = head * D, kx = (head / p.group) * D;
  auto load = [&](uint8_t* dst, int box, const CUtensorMap* map, int x, int y, uint32_t bar) {
#pragma unroll
    for (int b = 0; b < D / 64; ++b)
      tma_load_2d(smem_u32(dst + b * box), map, x + b * 64, y, bar);
  };
  if (warp == 8 && lane == 0) {
    mbar_init(smem_u32(q_full), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&kv_full[i]), 1);
      mbar_init(smem_u32(&kv_empty[i]), 1);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_full[i]), 4);
      mbar_init(smem_u32(&p_half[i]), 4);
      mbar_init(smem_u32(&pv_done[i]), 1);
    }
    mbar_init(smem_u32(drain), 1);
    *abort_flag = 0;
    fence_mbar_init();
    if (st.n > 0) {
      grid_wait();
      // the first loads run while tensor memory is allocated
      const uint32_t qb = smem_u32(q_full);
      mbar_expect_tx(qb, 2 * L::Q_BYTES + L::KV_BYTES);
      load(smem, L::Q_BOX, &p.tmap_q, qx, q_row, qb);
      load(smem + L::K_OFF, L::KV_BOX, &p.tmap_k, kx, k_row + st.base(0), qb);
      load(smem + L::Q_BYTES, L::Q_BOX, &p.tmap_q, qx, q_row + BQ, qb);
    }
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), L::TMEM_COLS);
    tmem_relinquish();
  }
  grid_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_launch_dependents();

  auto fail = [&]() {
    if (!*abort_flag) {
      record_error(H3B_ERR_TIMEOUT);
      *abort_flag = 1;
    }
  };

  // Each warpgroup changes its register limit inside its own branch and leaves
  // through its own copy of the teardown barrier.
  if (warp >= 8) {
    if constexpr (BK == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
    if (warp == 8) {
      if (lane == 0 && st.n > 0) {
        auto prefetch = [&](int j) {
          if (j < st.n) {
            const int y = k_row + st.base(j);
#pragma unroll
            for (int b = 0; b < D / 64; ++b) {
              tma_prefetch_2d(&p.tmap_k, kx + b * 64, y);
              tma_prefetch_2d(&p.tmap_v, kx + b * 64, y);
            }
          }
        };
        for (int j = 1; j < kPrefetchTiles; ++j) prefetch(j);
        int issued = 0;
        bool ok = true;
        for (int j = 0; j < st.n; ++j) {
          prefetch(j + kPrefetchTiles);
          if (j >= 1) {
            // release r = j - 2 frees K stage (j + 1) % 2 and V stage j % 2
            const int r = j - 2;
            const int s = r & 1;
            const int completion = s ? (r + 1) >> 1 : r >> 1;
            if (!mbar_wait(smem_u32(&kv_empty[s]), completion & 1, abort_flag)) {
              ok = false;
              break;
            }
          }
          const bool more = j + 1 < st.n;
          const uint32_t b = smem_u32(&kv_full[j & 1]);
          mbar_expect_tx(b, more ? 2 * L::KV_BYTES : L::KV_BYTES);
          load(smem + L::V_OFF + (j & 1) * L::KV_BYTES, L::KV_BOX, &p.tmap_v, kx,
               k_row + st.base(j), b);
          if (more)
            load(smem + L::K_OFF + ((j + 1) & 1) * L::KV_BYTES, L::KV_BOX, &p.tmap_k, kx,
                 k_row + st.base(j + 1), b);
          ++issued;
        }
        if (!ok) {
          // no copy may still be landing when the CTA exits
          fail();
          mbar_wait(smem_u32(q_full), 0, nullptr);
          for (int j = issued > 2 ? issued - 2 : 0; j < issued; ++j)
            mbar_wait(smem_u32(&kv_full[j & 1]), (j >> 1) & 1, nullptr);
        }
      }
    } else if (warp == 9 && st.n > 0) {
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort_flag));
      };
      const Range ra = tile_range(0), rb = tile_range(1);
      int last[2] = {-1, -1};
      for (int j = 0; j < st.n; ++j) {
        if (st.needed(ra, j)) last[0] = j;
        if (st.needed(rb, j)) last[1] = j;
      }
      auto need = [&](int t, int j) { return st.needed(t ? rb : ra, j); };
      auto issue_qk = [&](int t, int j) {
        const uint64_t qd = desc_kmajor_sw128(smem_u32(smem + t * L::Q_BYTES));
        const uint64_t kd = desc_kmajor_sw128(smem_u32(smem + L::K_OFF + (j & 1) * L::KV_BYTES));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)                // 16 head dims each
          tc_mma_bf16_ss_elect(tmem + L::s_col(t), qd + (((kk >> 2) * L::Q_BOX + (kk & 3) * 32) >> 4),
                               kd + (((kk >> 2) * L::KV_BOX + (kk & 3) * 32) >> 4), IDESC_QK,
                               kk != 0);
        tc_commit_elect(smem_u32(&s_full[t]));
      };
      int cnt[2] = {0, 0};                                 // needed steps done per tile
      auto pv_tile = [&](int t, int j) -> bool {
        // 16 keys per MMA: P columns kk * 8.. (pairs), V rows kk * 16.. (MN-major:
        // 64-dim chunks a box apart, 8-row groups 1 KiB)
        const uint64_t vd = smem_desc(smem_u32(smem + L::V_OFF + (j & 1) * L::KV_BYTES),
                                      L::KV_BOX, 1024, 2);
#pragma unroll
        for (int h = 0; h < L::HALVES; ++h) {
          if (!wait(h == L::HALVES - 1 ? &p_full[t] : &p_half[t], cnt[t] & 1)) return false;
          tc_fence_after();
#pragma unroll
          for (int kk = h * (L::P_FIRST / 16); kk < (h + 1 == L::HALVES ? BK : L::P_FIRST) / 16;
               ++kk) {
            tc_mma_bf16_ts_elect(tmem + L::o_col(t), tmem + L::s_col(t) + kk * 8,
                                 vd + kk * (2048 >> 4), IDESC_PV, (cnt[t] | kk) != 0);
          }
        }
        if (j == last[t]) tc_commit_elect(smem_u32(&pv_done[t]));
        ++cnt[t];
        return true;
      };
      bool ok = wait(q_full, 0);
      if (ok) {
        tc_fence_after();
        if (need(0, 0)) issue_qk(0, 0);
        if (need(1, 0)) issue_qk(1, 0);
        tc_commit_elect(smem_u32(&kv_empty[1]));           // release of K(0)
      }
      for (int j = 0; j < st.n && ok; ++j) {
        const bool more = j + 1 < st.n;
        if (!wait(&kv_full[j & 1], (j >> 1) & 1)) {
          ok = false;
          break;
        }
        const int valid = st.valid(j);
        if (valid < BK) {
          // V rows that no query sees: 8 chunks of 16 bytes per row and box
          uint8_t* v = smem + L::V_OFF + (j & 1) * L::KV_BYTES;
          for (int c = lane + valid * 8; c < BK * 8; c += 32) {
#pragma unroll
            for (int b = 0; b < D / 64; ++b)
              *reinterpret_cast<uint4*>(v + b * L::KV_BOX + c * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (need(t, j) && !pv_tile(t, j)) {
            ok = false;
            break;
          }
          if (more && need(t, j + 1)) issue_qk(t, j + 1);
        }
        if (ok) tc_commit_elect(smem_u32(&kv_empty[j & 1]));
      }
      if (!ok) {
        if (lane == 0) fail();
        tc_commit_elect(smem_u32(drain));
        mbar_wait(smem_u32(drain), 0, nullptr);
      }
    }
    tc_fence_before();
    named_barrier_sync(1, L::THREADS);
    if (warp == 9) {
      __syncwarp();
      tc_fence_after();
      tmem_dealloc(tmem, L::TMEM_COLS);
    }
  } else {
    if constexpr (BK == 128)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // softmax of tile t: thread = query row (TMEM lane quadrant warp % 4)
    const int t = warp >> 2;
    const int qd = warp & 3;
    const int r = qd * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(qd * 32) << 16;
    const uint32_t s_t = tmem + lane_addr + L::s_col(t);
    const uint32_t o_t = tmem + lane_addr + L::o_col(t);
    const Range rt = tile_range(t);
    const int pos = pos0 + t * BQ + r;                    // this row's key position
    const int w_first = pos0 + t * BQ + qd * 32;          // first and last position of the warp
    const int w_last = w_first + 31;
    const int top = p.causal ? pos : n_k - 1;             // last key the row may see
    const int w_top = p.causal ? w_first : n_k - 1;
    float m_used = -INFINITY, l = 0.f;
    int cnt = 0;
    bool ok = true;
    for (int j = 0; j < st.n; ++j) {
      if (!st.needed(rt, j)) continue;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[t]), cnt & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t sv[BK];
#pragma unroll
      for (int h = 0; h < BK / 64; ++h) tmem_ld_32x32b_x64(s_t + h * 64, sv + h * 64);
      tmem_ld_wait();
      const int base = st.base(j), valid = st.valid(j);
      const bool all_seen =                               // warp-uniform
          valid == BK && base + BK - 1 <= w_top &&
          (base + BK <= p.sinks || (base >= w_last - p.left && base + BK - 1 <= w_first + p.right));
      if (!all_seen) {
        const int a = pos - p.left - base;
        const int b = min(min(pos + p.right, top) - base, valid - 1);
        const int s = min(min(p.sinks - 1, top) - base, valid - 1);
#pragma unroll
        for (int w = 0; w < BK / 32; ++w) {
          const uint32_t seen = span_word(a, b, w) | span_word(0, s, w);
          if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (!(seen & (1u << c))) sv[w * 32 + c] = 0xff800000u;   // -inf: masked key
          }
        }
      }
      // row max of the scaled logits (scale > 0 commutes with max)
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < BK; c += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          m4[u] = attn::max3(m4[u], __uint_as_float(sv[c + 2 * u]), __uint_as_float(sv[c + 2 * u + 1]));
      }
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
      const float m_new = fmaxf(m_used, mx);
      if (__any_sync(0xffffffffu, m_new > m_used + attn::kRescaleLog2)) {
        // a row that has seen nothing yet stays at -inf (its l and O are 0)
        const float alpha = m_new == -INFINITY ? 1.f : attn::ex2(m_used - m_new);
        m_used = m_new;
        l *= alpha;
        if (cnt > 0) {
          // O is final up to the previous needed step: s_full of this one was
          // committed after its PV
#pragma unroll 1
          for (int h = 0; h < D / 16; ++h) {               // 16 at a time: S is in registers
            uint32_t ov[16];
            tmem_ld_x16(o_t + h * 16, ov);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 16; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
            tmem_st_x16(o_t + h * 16, ov);
          }
        }
      }
      float m = m_used == -INFINITY ? 0.f : m_used;         // -inf - (-inf) is no exponent
      float sc = p.scale_log2;
      // S * scale - m is one rounding of the exact product against a maximum that
      // was rounded before: the same for all keys of the row, so it cancels, but
      // from 2^27 on it reaches 2^3 and P its type's limit.  Then both are rounded.
      if (__any_sync(0xffffffffu, fabsf(m) > 16777216.f)) {
#pragma unroll
        for (int c = 0; c < BK; ++c)
          sv[c] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(sv[c]), sc), m));
        m = 0.f;
        sc = 1.f;
      }
      float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      softmax_store<T, 0, L::P_FIRST>(sv, sc, m, s_t, acc);
      if constexpr (L::HALVES == 2) {
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&p_half[t]));
        softmax_store<T, L::P_FIRST, BK - L::P_FIRST>(sv, sc, m, s_t, acc);
      }
      acc[0] = add2(acc[0], acc[1]);
      l += acc[0].x + acc[0].y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_full[t]));
      ++cnt;
    }
    if (ok && cnt > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&pv_done[t]), 0, abort_flag));
    if (!ok) fail();
    tc_fence_after();
    const int row = t * BQ + r;                            // of the pair's 256
    // does the row see any key at all
    const bool some = min(p.sinks, top + 1) > 0 ||
                      min(pos + p.right, min(top, n_k - 1)) >= max(0, pos - p.left);
    // The output leaves through the tile's Q buffer (all its MMAs are done), a
    // warp's 32 rows at a time: written a row per lane, 16-byte chunk c of row r
    // at chunk c ^ (r % 8), and copied out whole rows at a time.
    constexpr int CH = D / 8;                              // 16-byte chunks of a row
    uint4* const ostage = reinterpret_cast<uint4*>(smem + t * L::Q_BYTES) + qd * 32 * CH;
    auto stage = [&](int h, const uint32_t (&ov)[32], float inv_l) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          w[u] = some ? pack16<T>(__uint_as_float(ov[8 * c + 2 * u]) * inv_l,
                                  __uint_as_float(ov[8 * c + 2 * u + 1]) * inv_l)
                      : 0u;
        ostage[lane * CH + ((h * 4 + c) ^ (lane & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    // a part without a step of its own may have Q landing in that buffer still
    auto direct = [&](int h, const float (&acc)[32], float inv_l) {
      T* op = static_cast<T*>(p.out) + (size_t)(q_row + row) * p.ldo + (size_t)head * D + h * 32;
#pragma unroll
      for (int c = 0; c < 32; c += 2)
        *reinterpret_cast<uint32_t*>(op + c) =
            some ? pack16<T>(acc[c] * inv_l, acc[c + 1] * inv_l) : 0u;
    };
    auto copy_out = [&](bool zeros) {
      T* op = static_cast<T*>(p.out) + (size_t)(q_row + t * BQ + qd * 32) * p.ldo + (size_t)head * D;
      const int n = min(32, rows - t * BQ - qd * 32);      // rows of this warp
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * CH; i += 32) {
        const int rr = i / CH, c = i % CH;
        if (rr < n)
          *reinterpret_cast<uint4*>(op + (size_t)rr * p.ldo + c * 8) =
              zeros ? make_uint4(0, 0, 0, 0) : ostage[rr * CH + (c ^ (rr & 7))];
      }
    };
    if (whole) {
      const float inv_l = 1.0f / l;
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        if (ok && cnt > 0) {                               // warp-uniform
          uint32_t ov[32];
          tmem_ld_32x32b_x32(o_t + h * 32, ov);
          tmem_ld_wait();
          stage(h, ov, inv_l);
        }
      }
      if (ok) copy_out(cnt == 0);    // without a step Q may still be landing: zeros, no staging
    } else {
      // this part's O, m and l; the last part to arrive here adds all of them up
      constexpr int kPart = 256 * D + 512;                 // floats of a part
      float* mine = p.partial + ((size_t)split * p.parts + part) * kPart;
#pragma unroll
      for (int h = 0; h < D / 32; ++h) {
        uint32_t ov[32];
        if (ok && cnt > 0) {
          tmem_ld_32x32b_x32(o_t + h * 32, ov);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) ov[c] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 8; ++c)
          *reinterpret_cast<uint4*>(mine + ((h * 8 + c) * 256 + row) * 4) =
              make_uint4(ov[4 * c], ov[4 * c + 1], ov[4 * c + 2], ov[4 * c + 3]);
      }
      *reinterpret_cast<float2*>(mine + 256 * D + row * 2) = make_float2(m_used, l);
      __threadfence();
      named_barrier_sync(2, 256);
      volatile int* last = reinterpret_cast<volatile int*>(tmem_slot + 2);
      if (threadIdx.x == 0) {
        const bool is_last = atomicAdd(p.done + split, 1) == parts - 1;
        if (is_last) p.done[split] = 0;                    // for the next launch
        *last = is_last;
      }
      named_barrier_sync(2, 256);
      if (*last) {
        __threadfence();
        const float* all = p.partial + (size_t)split * p.parts * kPart;
        float mm = -INFINITY, ll = 0.f;
        for (int i = 0; i < parts; ++i)
          mm = fmaxf(mm, __ldcg(all + (size_t)i * kPart + 256 * D + row * 2));
        for (int i = 0; i < parts; ++i) {
          const float* ml = all + (size_t)i * kPart + 256 * D + row * 2;
          const float mi = __ldcg(ml);
          ll += mi == -INFINITY ? 0.f : attn::ex2(mi - mm) * __ldcg(ml + 1);
        }
        const float inv_l = 1.0f / ll;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          float acc[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[c] = 0.f;
          for (int i = 0; i < parts; ++i) {
            const float* from = all + (size_t)i * kPart;
            const float mi = __ldcg(from + 256 * D + row * 2);
            const float w = mi == -INFINITY ? 0.f : attn::ex2(mi - mm);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float4 v = __ldcg(
                  reinterpret_cast<const float4*>(from + ((h * 8 + c) * 256 + row) * 4));
              acc[4 * c] += w * v.x;
              acc[4 * c + 1] += w * v.y;
              acc[4 * c + 2] += w * v.z;
              acc[4 * c + 3] += w * v.w;
            }
          }
          if (cnt > 0) {
            uint32_t ov[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(acc[c]);
            stage(h, ov, inv_l);
          } else if (row < rows) {
            direct(h, acc, inv_l);
          }
        }
        if (cnt > 0) copy_out(false);
      }
    }
    tc_fence_before();
    named_barrier_sync(1, L::THREADS);
  }
}

}  // namespace wattn
}  // namespace h3b
