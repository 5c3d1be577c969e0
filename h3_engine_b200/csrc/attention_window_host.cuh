// Host side of the windowed-attention entry points (declared in include/h3b.h).
#pragma once

#include <cmath>

#include "attention_decode.cuh"
#include "attention_window.cuh"
#include "mx_host.cuh"

namespace h3b {

constexpr int64_t kMaxKeys = (int64_t)1 << 30;    // positions plus a window stay in 31 bits
constexpr int64_t kMaxGrid = 65535;               // along y and z

static inline int clamp_window(int64_t v) { return (int)std::min<int64_t>(v, kMaxKeys - 1); }

static int tmap_16_rows(CUtensorMap* tm, const void* base, int dtype, int64_t rows, int64_t cols,
                        int64_t stride, uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return H3B_ERR_UNSUPPORTED;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
  cuuint32_t box[2] = {64, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(tm, dtype == H3B_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? H3B_OK
             : H3B_ERR_INVALID_ARG;
}

template <int D, int BK, typename T>
static int window_attn_launch(const wattn::Args& a, int64_t grid, cudaStream_t st) {
  auto kernel = wattn::k_window_attn<D, BK, T>;
  using L = wattn::Cfg<D, BK>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  static SmemAttr attr;
  int rc = attr.set(fn, L::BYTES);
  if (rc != H3B_OK) return rc;
  if (BK == 128) {
    // the kernel's setmaxnreg split draws on this many launch registers
    static std::atomic<int> regs{0};
    if (!regs.load(std::memory_order_relaxed)) {
      cudaFuncAttributes fa;
      if (cudaFuncGetAttributes(&fa, fn) != cudaSuccess) return H3B_ERR_CUDA;
      regs.store(fa.numRegs, std::memory_order_relaxed);
    }
    if (regs.load(std::memory_order_relaxed) != wattn::kLaunchRegs) return H3B_ERR_UNSUPPORTED;
  }
  return launch(true, kernel, dim3((unsigned)grid), L::THREADS, L::BYTES, 0, st, a);
}

// Keys that an item of a document of n_k keys visits under a window.
static int64_t window_keys(int64_t n_k, int64_t left, int64_t right, int64_t sinks) {
  return std::min<int64_t>(n_k, left + right + 2 * wattn::BQ + sinks);
}

// One launch: up to MAX_DOCS documents with queries from d0 on, those with the
// most keys first (the light items then fill the last wave's gaps), and how
// their work is cut.
//   Items of 256 queries, or of 128 where those all have a place at once (1000
// rows, 8 heads: 17.9 us, in items of 256 19.5; 16384 rows, where they have
// not: 334 us, in items of 256 212), unless items of 256 can be cut into 3/2 as
// many parts.  The ratio lies between the cases measured: with as many parts
// items of 128 win as above, with twice as many items of 256 do (4000 rows, 2
// heads: 32.9 us, in items of 128 40.5).
//   Whole items first, then the last partial wave's in parts: items mod places
// would run alone, so they are split to fill the places (8 heads of 16384 rows,
// 512 items on 148 SMs: 212 us, unsplit 220).  A part keeps kPartKeys keys: the
// first split item, whose document has the most, says how many parts there are
// places for, and an item of fewer keys takes the first of them only (16 queries
// against 16000 keys beside a document of one key, one head: 64 us, 202 with as
// many parts for all as the fewest keys give).
struct WindowPlan {
  static constexpr int64_t kPartKeys = 512;
  int order[wattn::MAX_DOCS], doc_parts[wattn::MAX_DOCS];
  int n = 0, next = 0;
  int item_rows = 2 * wattn::BQ, step = 128, whole = 0, parts = 1;
  int64_t items = 0;
  WindowPlan(const int32_t* q_len, const int32_t* k_len, int ndocs, int d0, int H, int D,
             int64_t left, int64_t right, int64_t sinks) {
    for (; d0 < ndocs && n < wattn::MAX_DOCS; ++d0)
      if (q_len[d0] > 0) order[n++] = d0;
    next = d0;
    if (n == 0) return;
    std::sort(order, order + n, [&](int a, int b) {
      return k_len[a] != k_len[b] ? k_len[a] > k_len[b] : a < b;
    });
    auto count = [&](int rows) {
      int64_t c = 0;
      for (int i = 0; i < n; ++i) c += ((int64_t)q_len[order[i]] + rows - 1) / rows * H;
      return c;
    };
    const int sms = num_sms();
    auto doc_cut = [&](int i) {        // parts that a document's keys are enough for
      return std::max<int64_t>(1, window_keys(k_len[order[i]], left, right, sinks) / kPartKeys);
    };
    auto cut = [&](int64_t all, int rows, int places) {
      const int64_t rest = all % places;
      if (rest == 0) return (int64_t)1;
      int i = 0;                       // the document of the first split item
      for (int64_t end = 0;; ++i) {
        end += ((int64_t)q_len[order[i]] + rows - 1) / rows * H;
        if (end > all - rest) break;
      }
      return std::min<int64_t>(places / rest, doc_cut(i));
    };
    items = count(item_rows);
    if (const int64_t c = count(wattn::BQ);
        c <= sms && 2 * cut(items, item_rows, sms) < 3 * cut(c, wattn::BQ, sms)) {
      item_rows = wattn::BQ;
      items = c;
    }
    if (D == 64 && items > sms) step = 64;
    const int places = step == 64 ? 2 * sms : sms;
    parts = (int)cut(items, item_rows, places);
    whole = (int)std::min<int64_t>(parts > 1 ? items - items % places : items, INT32_MAX);
    for (int i = 0; i < n; ++i) doc_parts[i] = (int)std::min<int64_t>(parts, doc_cut(i));
  }
  int64_t split() const { return items - whole; }
  int64_t grid() const { return whole + split() * parts; }
};

static int64_t window_part_bytes(int D) { return ((int64_t)256 * D + 512) * 4; }
static constexpr int64_t kDoneBytes = 2048;       // a counter per split item (fewer than slots)

constexpr float kLog2e = 1.4426950408889634f;      // the kernels' exponents are of 2

static int window_rule(int64_t left, int64_t right, int64_t sinks, int causal, float scale) {
  if (left < 0 || right < 0 || sinks < 0 || (causal != 0 && causal != 1) || !(scale > 0.f) ||
      !std::isfinite(scale * kLog2e))
    return H3B_ERR_INVALID_ARG;
  return H3B_OK;
}

template <int D, typename T, int NT>
static int window_decode_rows(const wdec::Args& a, int64_t B, cudaStream_t st) {
  auto kernel = wdec::k_window_decode<D, T, NT>;
  constexpr int kBytes = wdec::Smem<D, NT>::BYTES;
  static SmemAttr attr;
  int rc = attr.set(reinterpret_cast<const void*>(kernel), kBytes);
  if (rc != H3B_OK) return rc;
  const int64_t row_tiles = ((int64_t)a.n_new * a.group + 8 * NT - 1) / (8 * NT);
  const int64_t groups = row_tiles * a.kv_heads;
  // CTAs along the keys: until there are two per SM, which run at a time (32
  // uneven sequences of 8 key heads: 91 us without a split, 76 with 512 CTAs,
  // 77 with 1024, 93 with 2048), but no more than give every warp two tiles
  // of a full window
  const int64_t most =
      std::min<int64_t>(a.room, (int64_t)a.left + a.right + a.n_new + (int64_t)a.sinks);
  int split = 1;
  while (split < wdec::kMaxCluster && groups * B * split < 2 * (int64_t)num_sms() &&
         most > (int64_t)split * wdec::kWarps * wdec::kKeys * 2)
    split *= 2;
  return launch(true, kernel, dim3((unsigned)split, (unsigned)groups, (unsigned)B), wdec::kThreads,
                      kBytes, split, st, a);
}

// Rows that share a key head: 8 of them in one product's columns, more in two.
template <int D, typename T>
static int window_decode_launch(const wdec::Args& a, int64_t B, cudaStream_t st) {
  return (int64_t)a.n_new * a.group <= 8 ? window_decode_rows<D, T, 1>(a, B, st)
                                         : window_decode_rows<D, T, 2>(a, B, st);
}

}  // namespace h3b

extern "C" {

int64_t h3b_attention_window_ws(const int32_t* q_len, const int32_t* k_len, int ndocs, int H,
                                int D, int64_t left, int64_t right, int64_t sinks) {
  if (!q_len || !k_len || ndocs <= 0 || H <= 0 || left < 0 || right < 0 || sinks < 0) return 0;
  left = clamp_window(left);
  right = clamp_window(right);
  sinks = clamp_window(sinks);
  int64_t most = 0;
  for (int d0 = 0; d0 < ndocs;) {
    const WindowPlan plan(q_len, k_len, ndocs, d0, H, D, left, right, sinks);
    d0 = plan.next;
    if (plan.n > 0 && plan.split() > 0)
      most = std::max(most, kDoneBytes + plan.split() * plan.parts * window_part_bytes(D));
  }
  return most;
}

int h3b_attention_window(const void* q, int64_t q_rows, int64_t q_stride, const void* k,
                         int64_t k_stride, const void* v, int64_t v_stride, int64_t kv_rows,
                         int dtype, int H, int kv_heads, int D, const int32_t* q_start,
                         const int32_t* q_len, const int32_t* k_start, const int32_t* k_len,
                         int ndocs, int64_t left, int64_t right, int64_t sinks, int causal,
                         float scale, void* out, int64_t ldo, void* ws, int64_t ws_bytes,
                         void* stream) {
  if (!dt_16(dtype) || (D != 64 && D != 128) || H <= 0 || kv_heads <= 0 || H % kv_heads ||
      ndocs < 0 || q_rows < 0 || kv_rows < 0)
    return H3B_ERR_INVALID_ARG;
  int rc = window_rule(left, right, sinks, causal, scale);
  if (rc != H3B_OK) return rc;
  const int64_t hd = (int64_t)H * D, kd = (int64_t)kv_heads * D;
  if (q_stride < hd || k_stride < kd || v_stride < kd || ldo < hd || hd > INT32_MAX)
    return H3B_ERR_INVALID_ARG;
  if (q_rows > kMaxKeys || kv_rows > kMaxKeys) return H3B_ERR_INVALID_ARG;
  if ((q_stride | k_stride | v_stride | ldo) % 8) return H3B_ERR_ALIGNMENT;
  if (ndocs > 0 && (!q_start || !q_len || !k_start || !k_len)) return H3B_ERR_INVALID_ARG;
  int64_t queries = 0, keys = 0;
  for (int i = 0; i < ndocs; ++i) {
    if (q_start[i] < 0 || q_len[i] < 0 || (int64_t)q_start[i] + q_len[i] > q_rows ||
        k_start[i] < 0 || k_len[i] < 0 || (int64_t)k_start[i] + k_len[i] > kv_rows)
      return H3B_ERR_INVALID_ARG;
    queries += q_len[i];
    keys += k_len[i];
  }
  if (queries == 0) return H3B_OK;
  if (!q || !out || (keys > 0 && (!k || !v))) return H3B_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return H3B_ERR_ALIGNMENT;
  rc = check_sm100();
  if (rc != H3B_OK) return rc;

  wattn::Args a;
  memset(&a, 0, sizeof(a));
  rc = tmap_16_rows(&a.tmap_q, q, dtype, q_rows, hd, q_stride, wattn::BQ);
  if (rc != H3B_OK) return rc;
  a.out = out;
  a.ldo = ldo;
  a.H = H;
  a.group = H / kv_heads;
  a.scale_log2 = scale * kLog2e;
  a.left = clamp_window(left);
  a.right = clamp_window(right);
  a.sinks = clamp_window(sinks);
  a.causal = causal;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t need =
      h3b_attention_window_ws(q_len, k_len, ndocs, H, D, left, right, sinks);
  if (need > 0) {
    if (!ws || ws_bytes < need) return H3B_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(ws) & 255u) return H3B_ERR_ALIGNMENT;
    if (cudaMemsetAsync(ws, 0, kDoneBytes, st) != cudaSuccess) return H3B_ERR_CUDA;
    a.done = static_cast<int*>(ws);
    a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kDoneBytes);
  }
  for (int d0 = 0; d0 < ndocs;) {               // documents in launches of MAX_DOCS
    const WindowPlan plan(q_len, k_len, ndocs, d0, H, D, a.left, a.right, a.sinks);
    d0 = plan.next;
    if (plan.n == 0) break;
    if (plan.items > INT32_MAX / 2) return H3B_ERR_INVALID_ARG;
    int64_t items = 0;
    for (int i = 0; i < plan.n; ++i) {
      const int d = plan.order[i];
      items += ((int64_t)q_len[d] + plan.item_rows - 1) / plan.item_rows * H;
      a.q_start[i] = q_start[d];
      a.q_len[i] = q_len[d];
      a.k_start[i] = k_start[d];
      a.k_len[i] = k_len[d];
      a.item_end[i] = (int)items;
      a.parts_of[i] = plan.doc_parts[i];
    }
    a.ndocs = plan.n;
    a.item_rows = plan.item_rows;
    a.whole = plan.whole;
    a.parts = plan.parts;
    // a step's keys are a box of the key and value maps
    if (keys > 0) {
      rc = tmap_16_rows(&a.tmap_k, k, dtype, kv_rows, kd, k_stride, (uint32_t)plan.step);
      if (rc != H3B_OK) return rc;
      rc = tmap_16_rows(&a.tmap_v, v, dtype, kv_rows, kd, v_stride, (uint32_t)plan.step);
      if (rc != H3B_OK) return rc;
    }
    auto go = [&](auto t) {
      using T = decltype(t);
      if (D == 128) return window_attn_launch<128, 128, T>(a, plan.grid(), st);
      if (plan.step == 128) return window_attn_launch<64, 128, T>(a, plan.grid(), st);
      return window_attn_launch<64, 64, T>(a, plan.grid(), st);
    };
    rc = dtype == H3B_DT_F16 ? go(__half()) : go(__nv_bfloat16());
    if (rc != H3B_OK) return rc;
  }
  return H3B_OK;
}

int h3b_attention_window_decode(const void* q, const int64_t* q_strides, const void* k,
                                const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                const int32_t* len, int64_t B, int64_t room, int64_t n_new,
                                int dtype, int H, int kv_heads, int D, int64_t left, int64_t right,
                                int64_t sinks, int causal, float scale, void* out, void* stream) {
  if (!dt_16(dtype) || (D != 64 && D != 128) || H <= 0 || kv_heads <= 0 || H % kv_heads || B < 0 ||
      room < 0 || n_new < 0 || room > kMaxKeys || n_new > kMaxGrid || !q_strides || !k_strides ||
      !v_strides)
    return H3B_ERR_INVALID_ARG;
  int rc = window_rule(left, right, sinks, causal, scale);
  if (rc != H3B_OK) return rc;
  for (int i = 0; i < 3; ++i) {
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 0) return H3B_ERR_INVALID_ARG;
    if ((q_strides[i] | k_strides[i] | v_strides[i]) % 8) return H3B_ERR_ALIGNMENT;
  }
  if (B == 0 || n_new == 0) return H3B_OK;
  if (!q || !len || !out || (room > 0 && (!k || !v))) return H3B_ERR_INVALID_ARG;
  // the grid's y and z
  if (B > kMaxGrid || (n_new * (H / kv_heads) + 15) / 16 * kv_heads > kMaxGrid)
    return H3B_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) ||
      (reinterpret_cast<uintptr_t>(len) & 3u))
    return H3B_ERR_ALIGNMENT;
  rc = check_sm100();
  if (rc != H3B_OK) return rc;
  wdec::Args a;
  memset(&a, 0, sizeof(a));
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.len = len;
  a.q_b = q_strides[0], a.q_t = q_strides[1], a.q_h = q_strides[2];
  a.k_b = k_strides[0], a.k_s = k_strides[1], a.k_h = k_strides[2];
  a.v_b = v_strides[0], a.v_s = v_strides[1], a.v_h = v_strides[2];
  a.room = (int)room;
  a.n_new = (int)n_new;
  a.H = H;
  a.kv_heads = kv_heads;
  a.group = H / kv_heads;
  a.left = clamp_window(left);
  a.right = clamp_window(right);
  a.sinks = clamp_window(sinks);
  a.causal = causal;
  a.scale_log2 = scale * kLog2e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D == 128)
    return dtype == H3B_DT_F16 ? window_decode_launch<128, __half>(a, B, st)
                               : window_decode_launch<128, __nv_bfloat16>(a, B, st);
  return dtype == H3B_DT_F16 ? window_decode_launch<64, __half>(a, B, st)
                             : window_decode_launch<64, __nv_bfloat16>(a, B, st);
}

}  // extern "C"
