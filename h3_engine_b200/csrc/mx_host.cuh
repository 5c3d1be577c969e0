// Host side of the MXFP4 entry points (declared in include/h3b.h): argument
// checks, TMA descriptors, kernel choice and launch.
#pragma once

#include "gemm_mxfp4.cuh"
#include "gemm_mxfp4_rows.cuh"
#include "quant_mx.cuh"

namespace h3b {

// Opt in a kernel's dynamic shared memory once per device (the attribute
// belongs to the device's context).
struct SmemAttr {
  std::atomic<bool> done[64];
  int set(const void* fn, int bytes) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return H3B_ERR_CUDA;
    if (dev < 64 && done[dev].load(std::memory_order_acquire)) return H3B_OK;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return H3B_ERR_CUDA;
    if (dev < 64) done[dev].store(true, std::memory_order_release);
    return H3B_OK;
  }
};

// One launch, as clusters of `cluster` CTAs along x.  early: it may come up
// under the end of the launch before it in the stream (common.cuh has the rules;
// one token against a cache of 4100 keys, calls in a row: 8.4 us, 10.4 as an
// ordinary launch).
template <typename... P, typename... A>
static int launch(bool early, void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster,
                  cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (early) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 0) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = 1;
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return launched(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// 2-D tensor of 16-bit values, box box_cols x box_rows, 128-byte swizzle.
static int make_tmap_16_sw128(CUtensorMap* map, const void* base, int dtype, uint64_t rows,
                              uint64_t cols, uint64_t pitch_elems, uint32_t box_cols,
                              uint32_t box_rows) {
  auto fn = encode_fn();
  if (!fn) return H3B_ERR_UNSUPPORTED;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {pitch_elems * 2};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, dtype == H3B_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? H3B_OK : H3B_ERR_INVALID_ARG;
}

static inline int dt_bytes(int dtype) { return dtype == H3B_DT_F32 ? 4 : 2; }
static inline bool dt_any(int d) { return d == H3B_DT_BF16 || d == H3B_DT_F16 || d == H3B_DT_F32; }
static inline bool dt_16(int d) { return d == H3B_DT_BF16 || d == H3B_DT_F16; }

constexpr int64_t kMxMaxDim = (int64_t)INT32_MAX - 512;

// One unit of work per warp (32768 x 14336 bf16: 207 and 226 us to quantize and
// unpack with 8 CTAs per SM that loop, 176 and 190 with 32, 177 and 177 with as
// many as there are units), two loads in flight per lane (one: 186 and 187).
constexpr int kQuantUnroll = 2;
static unsigned mx_quant_blocks(int64_t units) {
  const int64_t blocks = (units + mx::kThreads / 32 - 1) / (mx::kThreads / 32);
  return (unsigned)std::min<int64_t>(blocks, 1 << 30);
}

template <typename T, int VPL>
static int mx_quantize_launch(const void* x, int64_t M, int64_t K, int64_t ldx, void* q,
                              int64_t ldq, void* sf, cudaStream_t st) {
  constexpr int kUnit = 32 * VPL * kQuantUnroll;
  const int64_t Mpad = (M + 127) / 128 * 128;
  const int64_t per_row = (mx::sf_tiles(K) * 128 + kUnit - 1) / kUnit;
  return launch(true, mx::k_mxfp4_quantize<T, VPL, kQuantUnroll>,
                      dim3(mx_quant_blocks(Mpad * per_row)), mx::kThreads, 0, 0, st,
                      static_cast<const T*>(x), M, K, ldx, static_cast<uint8_t*>(q), ldq,
                      static_cast<uint8_t*>(sf), Mpad, (uint32_t)per_row);
}

template <typename T, int VPL>
static int mx_dequantize_launch(const void* q, const void* sf, int64_t M, int64_t K, void* out,
                                int64_t ldo, cudaStream_t st) {
  constexpr int kUnit = 32 * VPL * kQuantUnroll;
  const int64_t per_row = (K + kUnit - 1) / kUnit;
  return launch(true, mx::k_mxfp4_dequantize<T, VPL, kQuantUnroll>,
                      dim3(mx_quant_blocks(M * per_row)), mx::kThreads, 0, 0, st,
                      static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(sf), M, K,
                      static_cast<T*>(out), ldo, (uint32_t)per_row);
}

// 32-byte accesses where base and rows allow them.
static inline bool wide_rows(const void* p, int64_t ld, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 31u) == 0 && (ld * size) % 32 == 0;
}

static int mx_quantize(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, void* q,
                       int64_t ldq, void* sf, cudaStream_t st) {
  if (!dt_any(dtype) || M < 0 || K <= 0 || K % mx::BLOCK || ldx < K) return H3B_ERR_INVALID_ARG;
  if (M > kMxMaxDim || K > kMxMaxDim) return H3B_ERR_INVALID_ARG;
  if (M == 0) return H3B_OK;
  if (!x || !q || !sf) return H3B_ERR_INVALID_ARG;
  if (!aligned16(x) || !aligned16(q) || !aligned16(sf) || (ldx * dt_bytes(dtype)) % 16)
    return H3B_ERR_ALIGNMENT;
  const bool wide = wide_rows(x, ldx, dt_bytes(dtype));
  auto go = [&](auto t) {
    using T = decltype(t);
    return wide ? mx_quantize_launch<T, 16>(x, M, K, ldx, q, ldq, sf, st)
                : mx_quantize_launch<T, 8>(x, M, K, ldx, q, ldq, sf, st);
  };
  if (dtype == H3B_DT_BF16) return go(__nv_bfloat16());
  if (dtype == H3B_DT_F16) return go(__half());
  return go(float());
}

// Operands of the CTA-pair kernel: shapes and alignment.
static int mx_gemm_args(mxgemm::PairArgs& pa, const void* A, int64_t lda, const void* sfA,
                        int64_t M, const void* B, const void* sfB, int64_t N, int64_t K) {
  if (!A || !sfA || !B || !sfB) return H3B_ERR_INVALID_ARG;
  if (!aligned16(A) || !aligned16(sfA) || !aligned16(B) || !aligned16(sfB))
    return H3B_ERR_ALIGNMENT;
  int rc = check_sm100();
  if (rc != H3B_OK) return rc;
  memset(&pa, 0, sizeof(pa));
  mxgemm::Args& a = pa.base;
  rc = make_tmap_u8_sw128(&a.tmap_a, A, (uint64_t)M, (uint64_t)(K / 2), (uint64_t)lda,
                          mxgemm::KB_BYTES, mxgemm::BM);
  if (rc != H3B_OK) return rc;
  rc = make_tmap_u8_sw128(&a.tmap_b, B, (uint64_t)N, (uint64_t)(K / 2), (uint64_t)(K / 2),
                          mxgemm::KB_BYTES, 128);
  if (rc != H3B_OK) return rc;
  a.sfa = static_cast<const uint8_t*>(sfA);
  a.sfb = static_cast<const uint8_t*>(sfB);
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.sf_tiles_k = (int)mx::sf_tiles(K);
  a.n_tiles = (int)((N + mxgemm::BN - 1) / mxgemm::BN);
  pa.m_tiles = (int)((M + 255) / 256);
  if ((int64_t)pa.m_tiles * a.n_tiles > INT32_MAX) return H3B_ERR_INVALID_ARG;
  const uint64_t width = (uint64_t)a.sf_tiles_k * (mxgemm::SF_ATOM / 8);
  rc = make_tmap_u64(&pa.tmap_sfa, sfA, (uint64_t)((M + 127) / 128), width, mxgemm::KB_ATOMS * 64,
                     1);
  if (rc != H3B_OK) return rc;
  rc = make_tmap_u64(&pa.tmap_sfb, sfB, (uint64_t)((N + 127) / 128), width, mxgemm::KB_ATOMS * 64,
                     2);
  if (rc != H3B_OK) return rc;
  // 16 tile rows per raster group: the 74 pairs then work on 16 row and about
  // 5 column tiles at a time (13383 x 28672 x 5376: 889 us with groups of one,
  // 843 of 4, 811 of 8, 793 of 16, 784 of 32; shorter N, 193-198)
  pa.group = 16;
  return H3B_OK;
}

// chained: the launch before is of the same call, and the weight does not wait
// for it (a product alone is an ordinary launch).  The next launch comes up under
// a product in a chain (the feed-forward's up projection), and under one of a
// single wave of tiles (1025 rows through 2016 x 5504 and back: 31.1 us, else
// 33.0); under a longer one it costs more than the launch (13383 x 5376 x 7168
// with its quantization: 237 us, else 231).
template <typename T, int EPI>
static int mx_gemm_launch(mxgemm::PairArgs& pa, bool chained, cudaStream_t st) {
  auto kernel = mxgemm::k_gemm_mxfp4_pair<T, EPI>;
  static SmemAttr attr;
  const int rc = attr.set(reinterpret_cast<const void*>(kernel), mxgemm::P_SMEM_BYTES);
  if (rc != H3B_OK) return rc;
  const int64_t tiles = (int64_t)pa.m_tiles * pa.base.n_tiles;
  const int pairs = (int)std::min<int64_t>(tiles, num_sms() / 2);
  pa.base.early = EPI == mxgemm::kSwigluQuant || tiles <= pairs;
  return launch(chained, kernel, dim3((unsigned)(2 * pairs)), mxgemm::THREADS,
                mxgemm::P_SMEM_BYTES, 0, st, pa);
}

// ---- up to 128 rows: the weight-streaming kernel
constexpr int64_t kRowsMaxN = (int64_t)65535 * mxrows::BN;    // weight tiles are its grid's y

// CTAs along K, a power of two of them (clusters of odd sizes do not all find
// room at once): while two per SM hold them all and two k-blocks are left to
// each (1 x 7168 x 5376: 9.1 us on one, 7.3 on two, 6.9 on four; 77 x 4136 x
// 2720: 11.5, 9.5, 8.5 and, with one k-block each on eight, 9.6)
static int mx_rows_split(int64_t tiles, int64_t K) {
  const int64_t num_kb = (K + mxrows::KB_ELEMS - 1) / mxrows::KB_ELEMS;
  int split = 1;
  while (split * 2 <= mxrows::kMaxSplit && split * 2 * tiles <= 2 * num_sms() &&
         num_kb >= split * 4)
    split *= 2;
  return split;
}

// Does the product quantize its rows itself: up to 8, and up to 32 where that is
// at most two units of 8 rows and a k-block for each of a CTA's four warps (16 x
// 2048 x 2048, one unit: 4.5 us on the device, 5.1 with a launch of its own; 32 x
// 2048 x 2048, two: 5.8 and 5.5, but calls in a row are bound by their launches,
// 7.6 and 10.4; past that 16 x 7168 x 5376: 10.6 and 8.8).
static bool mx_fused(int64_t M, int64_t N, int64_t K) {
  if (M > mxrows::kFusedRows || N > kRowsMaxN) return false;
  if (M <= mxrows::kUnitRows) return true;
  const int split = mx_rows_split((N + mxrows::BN - 1) / mxrows::BN, K);
  const int64_t kbs = ((K + mxrows::KB_ELEMS - 1) / mxrows::KB_ELEMS + split - 1) / split;
  return kbs * ((M + mxrows::kUnitRows - 1) / mxrows::kUnitRows) <= 8;
}

template <int MT, typename T, int EPI, int FUSED>
static int mx_rows_launch(mxrows::Args& a, const void* A, const void* B, bool chained,
                          cudaStream_t st) {
  a.first = !chained;
  int rc = make_tmap_u8_sw128(&a.tmap_w, B, (uint64_t)a.N, (uint64_t)(a.K / 2),
                              (uint64_t)(a.K / 2), mxrows::KB_BYTES, mxrows::BN);
  if (rc != H3B_OK) return rc;
  if (!FUSED) {
    rc = make_tmap_u8_sw128(&a.tmap_x, A, (uint64_t)a.M, (uint64_t)(a.K / 2), (uint64_t)a.ldx,
                            mxrows::KB_BYTES, MT);
    if (rc != H3B_OK) return rc;
  }
  auto kernel = mxrows::k_gemm_mxfp4_rows<MT, T, EPI, FUSED>;
  static SmemAttr attr;
  rc = attr.set(reinterpret_cast<const void*>(kernel), mxrows::Ring<MT>::BYTES);
  if (rc != H3B_OK) return rc;
  const int tiles = (a.N + mxrows::BN - 1) / mxrows::BN;
  const int m_tiles = (a.M + MT - 1) / MT;      // more than one only for MT = 128
  const int split = mx_rows_split((int64_t)tiles * m_tiles, a.K);
  return launch(true, kernel, dim3((unsigned)split, (unsigned)tiles, (unsigned)m_tiles),
                      mxrows::THREADS, mxrows::Ring<MT>::BYTES, split, st, a);
}

// Operands of the rows kernel: A as codes (ldx bytes a row) and scales, or (sfA
// NULL) as 16-bit rows of ldx elements that the kernel quantizes itself.
template <typename T, int EPI>
static int mx_rows_gemm(mxrows::Args& a, const void* A, const void* sfA, int64_t ldx, int64_t M,
                        const void* B, const void* sfB, int64_t N, int64_t K, bool chained,
                        cudaStream_t st) {
  if (!A || !B || !sfB) return H3B_ERR_INVALID_ARG;
  if (!aligned16(A) || !aligned16(sfA) || !aligned16(B) || !aligned16(sfB))
    return H3B_ERR_ALIGNMENT;
  const int rc = check_sm100();
  if (rc != H3B_OK) return rc;
  a.sfw = static_cast<const uint8_t*>(sfB);
  a.sfx = static_cast<const uint8_t*>(sfA);
  a.x = A;
  a.ldx = ldx;
  a.M = (int)M;
  a.N = (int)N;
  a.K = (int)K;
  a.sf_tiles_k = (int)mx::sf_tiles(K);
  if (!sfA)
    return M <= mxrows::kUnitRows ? mx_rows_launch<16, T, EPI, 1>(a, A, B, chained, st)
           : M <= 16              ? mx_rows_launch<16, T, EPI, 2>(a, A, B, chained, st)
                                  : mx_rows_launch<32, T, EPI, 2>(a, A, B, chained, st);
  if (M <= 16) return mx_rows_launch<16, T, EPI, 0>(a, A, B, chained, st);
  if (M <= 32) return mx_rows_launch<32, T, EPI, 0>(a, A, B, chained, st);
  if (M <= 64) return mx_rows_launch<64, T, EPI, 0>(a, A, B, chained, st);
  return mx_rows_launch<128, T, EPI, 0>(a, A, B, chained, st);
}

// An activation's codes are ours to lay out: rows start at whole sectors (32
// bytes), so that a TMA box's rows take no sector more than they fill (13383 x
// 4096 x 4064 with its quantization: 114 us, 122 with rows of K / 2 bytes; 1025 x
// 11008 x 2016: 19.0 and 20.3).
static inline int64_t mx_code_pitch(int64_t k) { return (k / 2 + 31) / 32 * 32; }
// Bytes of them in a workspace, rounded up to 256, and with their blocked scales.
static inline int64_t mx_code_bytes(int64_t rows, int64_t k) {
  return (rows * mx_code_pitch(k) + 255) / 256 * 256;
}
static inline int64_t mx_operand_bytes(int64_t rows, int64_t k) {
  return mx_code_bytes(rows, k) + (rows + 127) / 128 * mx::sf_tiles(k) * mxgemm::SF_ATOM;
}

// Checks of everything but the operands of a product D = act(A B^T + bias) + residual.
static int mx_out_check(int dtype, int64_t M, int64_t N, int64_t K, const void* bias, int act,
                        const void* residual, int64_t ldr, const void* D, int64_t ldd) {
  if (!dt_16(dtype) || M < 0 || N <= 0 || K <= 0 || K % mx::BLOCK || N % 8) return H3B_ERR_INVALID_ARG;
  if (act != H3B_ACT_NONE && act != H3B_ACT_GELU_TANH) return H3B_ERR_INVALID_ARG;
  if (M > kMxMaxDim || N > kMxMaxDim || K > kMxMaxDim) return H3B_ERR_INVALID_ARG;
  if (ldd < N || (residual && ldr < N)) return H3B_ERR_INVALID_ARG;
  if (M == 0) return H3B_OK;
  if (!D) return H3B_ERR_INVALID_ARG;
  if (ldd % 8 || (residual && ldr % 8) || !aligned16(D) || (bias && !aligned16(bias)) ||
      (residual && !aligned16(residual)))
    return H3B_ERR_ALIGNMENT;
  return H3B_OK;
}

// Which kernel: the rows kernel (whose grid takes N up to kRowsMaxN) up to 128
// rows, and beyond them in tiles of 128
// where the pair kernel would leave most SMs idle over a long K: where three
// CTAs along K find room for each of its tiles (144 x 2048 x 5376: 11.1 us
// against 13.5, 512 x 2048 x 5376: 12.8 and 13.4, 256 x 5376 x 14336: 22.3 and
// 26.9; past that 512 x 5376 x 14336: 34.1 and 28.7; with K = 2048 the pair
// kernel is ahead, 256 x 5376: 11.2 and 9.5).
static bool mx_by_rows(int64_t M, int64_t N, int64_t K) {
  return N <= kRowsMaxN &&
         (M <= mxrows::kMaxRows ||
          (K >= 4096 && ((M + 127) / 128) * ((N + 127) / 128) * 3 <= 2 * num_sms()));
}

// D = act(A B^T + bias) + residual.  A is codes, ldx bytes a row, or (sfA NULL,
// mx_fused) 16-bit rows of ldx elements.  chained: the launch before is of the same entry point.
static int mx_gemm_out(const void* A, const void* sfA, int64_t ldx, int64_t M, const void* B,
                       const void* sfB, int64_t N, int64_t K, const void* bias, int act,
                       const void* residual, int64_t ldr, void* D, int dtype, int64_t ldd,
                       bool chained, cudaStream_t st) {
  ldr = residual ? ldr : 0;
  if (mx_by_rows(M, N, K)) {
    mxrows::Args a;
    memset(&a, 0, sizeof(a));
    a.bias = bias;
    a.residual = residual;
    a.out = D;
    a.ldr = ldr;
    a.ldd = ldd;
    a.act = act;
    return dtype == H3B_DT_F16
               ? mx_rows_gemm<__half, mxgemm::kOut>(a, A, sfA, ldx, M, B, sfB, N, K, chained, st)
               : mx_rows_gemm<__nv_bfloat16, mxgemm::kOut>(a, A, sfA, ldx, M, B, sfB, N, K,
                                                           chained, st);
  }
  mxgemm::PairArgs pa;
  int rc = mx_gemm_args(pa, A, ldx, sfA, M, B, sfB, N, K);
  if (rc != H3B_OK) return rc;
  mxgemm::Args& a = pa.base;
  rc = make_tmap_16_sw128(&a.tmap_d, D, dtype, (uint64_t)M, (uint64_t)N, (uint64_t)ldd,
                          mxgemm::OUT_COLS, 32);
  if (rc != H3B_OK) return rc;
  a.bias = bias;
  if (residual) {
    rc = make_tmap_16_sw128(&a.tmap_r, residual, dtype, (uint64_t)M, (uint64_t)N, (uint64_t)ldr,
                            mxgemm::OUT_COLS, 32);
    if (rc != H3B_OK) return rc;
    a.residual = 1;
  }
  if (act == H3B_ACT_GELU_TANH)
    return dtype == H3B_DT_F16
               ? mx_gemm_launch<__half, mxgemm::kOutGelu>(pa, chained, st)
               : mx_gemm_launch<__nv_bfloat16, mxgemm::kOutGelu>(pa, chained, st);
  return dtype == H3B_DT_F16 ? mx_gemm_launch<__half, mxgemm::kOut>(pa, chained, st)
                             : mx_gemm_launch<__nv_bfloat16, mxgemm::kOut>(pa, chained, st);
}

// 16-bit rows that a product can quantize itself.
static int mx_input_check(const void* x, int64_t ldx, int64_t K) {
  if (!x || ldx < K) return H3B_ERR_INVALID_ARG;
  return !aligned16(x) || ldx % 8 ? H3B_ERR_ALIGNMENT : H3B_OK;
}

}  // namespace h3b

extern "C" {

int h3b_mxfp4_quantize(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, void* q,
                       void* sf, void* stream) {
  return mx_quantize(x, dtype, M, K, ldx, q, K / 2, sf, static_cast<cudaStream_t>(stream));
}

int h3b_mxfp4_dequantize(const void* q, const void* sf, int64_t M, int64_t K, void* out, int dtype,
                         int64_t ldo, void* stream) {
  if (!dt_any(dtype) || M < 0 || K <= 0 || K % mx::BLOCK || ldo < K) return H3B_ERR_INVALID_ARG;
  if (M > kMxMaxDim || K > kMxMaxDim) return H3B_ERR_INVALID_ARG;
  if (M == 0) return H3B_OK;
  if (!q || !sf || !out) return H3B_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(out) || (ldo * dt_bytes(dtype)) % 16) return H3B_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = wide_rows(out, ldo, dt_bytes(dtype));
  auto go = [&](auto t) {
    using T = decltype(t);
    return wide ? mx_dequantize_launch<T, 16>(q, sf, M, K, out, ldo, st)
                : mx_dequantize_launch<T, 8>(q, sf, M, K, out, ldo, st);
  };
  if (dtype == H3B_DT_BF16) return go(__nv_bfloat16());
  if (dtype == H3B_DT_F16) return go(__half());
  return go(float());
}

int h3b_mxfp4_gemm(const void* A, const void* sfA, int64_t M, const void* B, const void* sfB,
                   int64_t N, int64_t K, const void* bias, int act, const void* residual,
                   int64_t ldr, void* D, int dtype, int64_t ldd, void* stream) {
  const int rc = mx_out_check(dtype, M, N, K, bias, act, residual, ldr, D, ldd);
  if (rc != H3B_OK || M == 0) return rc;
  if (!sfA) return H3B_ERR_INVALID_ARG;
  return mx_gemm_out(A, sfA, K / 2, M, B, sfB, N, K, bias, act, residual, ldr, D, dtype, ldd, false,
                     static_cast<cudaStream_t>(stream));
}

int64_t h3b_mxfp4_linear_ws(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kMxMaxDim || K > kMxMaxDim) return 0;
  if (M <= mxrows::kUnitRows && N <= kRowsMaxN) return 0;
  return mx_operand_bytes(M, K);
}

int h3b_mxfp4_linear(const void* x, int dtype, int64_t M, int64_t ldx, const void* B,
                     const void* sfB, int64_t N, int64_t K, const void* bias, int act,
                     const void* residual, int64_t ldr, void* D, int64_t ldd, void* ws,
                     int64_t ws_bytes, void* stream) {
  int rc = mx_out_check(dtype, M, N, K, bias, act, residual, ldr, D, ldd);
  if (rc != H3B_OK || M == 0) return rc;
  const int64_t need = h3b_mxfp4_linear_ws(M, N, K);
  if (need > 0 && (!ws || ws_bytes < need)) return H3B_ERR_INVALID_ARG;
  if (need > 0 && reinterpret_cast<uintptr_t>(ws) & 255u) return H3B_ERR_ALIGNMENT;
  rc = mx_input_check(x, ldx, K);
  if (rc != H3B_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (mx_fused(M, N, K))
    return mx_gemm_out(x, nullptr, ldx, M, B, sfB, N, K, bias, act, residual, ldr, D, dtype, ldd,
                       false, st);
  uint8_t* q = static_cast<uint8_t*>(ws);
  uint8_t* sf = q + mx_code_bytes(M, K);
  const int64_t pitch = mx_code_pitch(K);
  rc = mx_quantize(x, dtype, M, K, ldx, q, pitch, sf, st);
  if (rc != H3B_OK) return rc;
  return mx_gemm_out(q, sf, pitch, M, B, sfB, N, K, bias, act, residual, ldr, D, dtype, ldd, true, st);
}

int64_t h3b_mxfp4_ffn_ws(int64_t M, int64_t N, int64_t F) {
  if (M < 0 || N <= 0 || F <= 0 || M > kMxMaxDim || N > kMxMaxDim || F > kMxMaxDim) return 0;
  return mx_operand_bytes(M, N) + mx_operand_bytes(M, F);
}

int h3b_mxfp4_ffn(const void* x, int dtype, int64_t M, int64_t ldx, const void* Bu,
                  const void* sfBu, const void* Bd, const void* sfBd, int64_t N, int64_t F,
                  const void* residual, int64_t ldr, void* D, int64_t ldd, void* ws,
                  int64_t ws_bytes, void* stream) {
  if (F <= 0 || F % 128 || F > kMxMaxDim / 2 || N % mx::BLOCK) return H3B_ERR_INVALID_ARG;
  int rc = mx_out_check(dtype, M, N, F, nullptr, H3B_ACT_NONE, residual, ldr, D, ldd);
  if (rc != H3B_OK || M == 0) return rc;
  if (!ws || ws_bytes < h3b_mxfp4_ffn_ws(M, N, F)) return H3B_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return H3B_ERR_ALIGNMENT;
  rc = mx_input_check(x, ldx, N);
  if (rc != H3B_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* q = static_cast<uint8_t*>(ws);
  uint8_t* sf = q + mx_code_bytes(M, N);
  uint8_t* qh = q + mx_operand_bytes(M, N);
  uint8_t* sfh = qh + mx_code_bytes(M, F);
  const bool fused = mx_fused(M, 2 * F, N);
  const int64_t pitch = mx_code_pitch(N);
  if (!fused) {
    rc = mx_quantize(x, dtype, M, N, ldx, q, pitch, sf, st);
    if (rc != H3B_OK) return rc;
  }
  if (mx_by_rows(M, 2 * F, N)) {
    mxrows::Args a;
    memset(&a, 0, sizeof(a));
    a.q_out = qh;
    a.sf_out = sfh;
    const void* A = fused ? x : q;
    const void* sfA = fused ? nullptr : sf;
    const int64_t lda = fused ? ldx : pitch;
    rc = dtype == H3B_DT_F16
             ? mx_rows_gemm<__half, mxgemm::kSwigluQuant>(a, A, sfA, lda, M, Bu, sfBu, 2 * F, N,
                                                          !fused, st)
             : mx_rows_gemm<__nv_bfloat16, mxgemm::kSwigluQuant>(a, A, sfA, lda, M, Bu, sfBu,
                                                                 2 * F, N, !fused, st);
  } else {
    mxgemm::PairArgs up;
    rc = mx_gemm_args(up, q, pitch, sf, M, Bu, sfBu, 2 * F, N);
    if (rc != H3B_OK) return rc;
    up.base.q_out = qh;
    up.base.sf_out = sfh;
    rc = mx_gemm_launch<__nv_bfloat16, mxgemm::kSwigluQuant>(up, true, st);
  }
  if (rc != H3B_OK) return rc;
  return mx_gemm_out(qh, sfh, F / 2, M, Bd, sfBd, N, F, nullptr, H3B_ACT_NONE, residual, ldr, D,
                     dtype, ldd, true, st);
}

}  // extern "C"
