// torch operators (namespace h3b) of the MXFP4 and windowed-attention entry
// points, in C++: these serve single tokens, where an operator written in
// Python costs several times the kernel it launches.  Each checks its tensors
// (ValueError, TypeError), allocates results and workspaces from torch's
// caching allocator, and calls the C ABI of libh3b.so on the current stream of
// its tensors' device.  Only CUDA implementations are registered.  Built as
// _h3b_torch.so beside libh3b.so, which it links.
#include <ATen/ATen.h>
#include <ATen/TensorUtils.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>
#include <vector>

#include "h3b.h"

namespace {

using at::Tensor;
using std::optional;

void check(int status, const char* what) {
  TORCH_CHECK(status == H3B_OK, what, " failed: status ", status, " (", h3b_status_string(status),
              ")");
}

// The call's device, current stream and guard; every tensor has to live there.
struct Call {
  c10::cuda::CUDAGuard guard;
  c10::Device dev;
  explicit Call(const Tensor& t) : guard(on_cuda(t)), dev(t.device()) {}
  static c10::Device on_cuda(const Tensor& t) {
    TORCH_CHECK_VALUE(t.is_cuda(), "h3b ops take CUDA tensors (there is no CPU path)");
    return t.device();
  }
  void same(const Tensor& t) const {
    TORCH_CHECK_VALUE(t.device() == dev, "tensors on different devices: ", dev, " vs ", t.device());
  }
  void same(const optional<Tensor>& t) const {
    if (t) same(*t);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }
};

int dtype_code(const Tensor& t, bool f32_too, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return H3B_DT_BF16;
    case at::kHalf: return H3B_DT_F16;
    case at::kFloat:
      if (f32_too) return H3B_DT_F32;
      break;
    default: break;
  }
  TORCH_CHECK_TYPE(false, what, " takes ", f32_too ? "bf16, fp16 or fp32" : "bf16 or fp16",
                   ", not ", t.scalar_type());
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool rows_aligned(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) >= t.size(1) &&
         t.stride(0) * (int64_t)t.element_size() % 16 == 0 && aligned(t.data_ptr());
}

// A [rows, C] view with contiguous, 16-byte aligned rows (a copy only when the
// layout needs one).
Tensor rows2d(const Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() >= 1, "a tensor of rows is expected");
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return rows_aligned(r) ? r : r.clone(at::MemoryFormat::Contiguous);
}

// New tensors straight from the caching allocator (no dispatch).
Tensor new_tensor(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(shape, type, like.device(), std::nullopt);
}
Tensor scratch(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? new_tensor({bytes}, at::kByte, like) : Tensor();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

int64_t sf_bytes(int64_t rows, int64_t k) { return (rows + 127) / 128 * ((k + 127) / 128) * 512; }

void check_operand(const Tensor& q, const Tensor& sf, int64_t rows, int64_t k, const char* what) {
  TORCH_CHECK_TYPE(q.scalar_type() == at::kByte && sf.scalar_type() == at::kByte, what,
                   ": codes and scales must be uint8");
  TORCH_CHECK_VALUE(k > 0 && k % 32 == 0, what, ": K = ", k, " must be a positive multiple of 32");
  TORCH_CHECK_VALUE(rows >= 0, what, ": negative row count");
  TORCH_CHECK_VALUE(q.is_contiguous() && sf.is_contiguous(), what,
                    ": codes and scales must be contiguous");
  TORCH_CHECK_VALUE(q.numel() >= rows * (k / 2) && sf.numel() >= sf_bytes(rows, k), what,
                    ": codes or scales too small for ", rows, " x ", k, " values");
  TORCH_CHECK_VALUE(aligned(q.data_ptr()) && aligned(sf.data_ptr()), what,
                    ": codes and scales must be 16-byte aligned");
}

void check_n(int64_t n) {
  TORCH_CHECK_VALUE(n > 0 && n % 8 == 0, "N = ", n, " must be a positive multiple of 8");
}

Tensor new_out(const Tensor& like, int64_t n, at::ScalarType type) {
  auto shape = like.sizes().vec();
  shape.back() = n;
  return new_tensor(shape, type, like);
}

// A tensor's bytes: from `at`, up to `end`, and, where its leading dimensions
// are evenly spaced, as `rows` rows of `width` bytes every `pitch`.
struct Bytes {
  uintptr_t at, end;
  int64_t rows = 1, width, pitch = 0;
  bool even;
  explicit Bytes(const Tensor& t) : at(reinterpret_cast<uintptr_t>(t.data_ptr())) {
    const int64_t size = t.element_size();
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    end = at + (last + 1) * size;
    const int64_t cols = t.dim() ? t.size(-1) : 1;
    width = cols * size;
    even = t.dim() == 0 || cols == 1 || t.stride(-1) == 1;
    for (int64_t i = t.dim() - 2; i >= 0; --i) {
      if (t.size(i) == 1) continue;
      if (rows == 1) pitch = t.stride(i) * size;
      else even = even && t.stride(i) * size == pitch * rows;
      rows *= t.size(i);
    }
    if (rows > 1 && pitch == width) {              // no gaps: one row
      width *= rows;
      rows = 1;
    }
  }
};

// An output may be one of its inputs where every element is read before it is
// written by the same thread (exact_ok), and shares no memory with the others;
// columns side by side in the same rows share none.
void apart(const Tensor& out, const Tensor& in, bool exact_ok, const char* what) {
  if (out.numel() == 0 || in.numel() == 0) return;
  const Bytes a(out), b(in);
  if (a.end <= b.at || b.end <= a.at) return;
  bool ok = false;
  if (a.even && b.even) {
    if (a.at == b.at && a.rows == b.rows && a.width == b.width && a.pitch == b.pitch) {
      ok = exact_ok;
    } else if (a.rows > 1 && b.rows > 1 && a.pitch == b.pitch && a.pitch > 0) {
      const Bytes &lo = a.at < b.at ? a : b, &hi = a.at < b.at ? b : a;
      const int64_t d = (int64_t)(hi.at - lo.at) % a.pitch;
      ok = d >= lo.width && d + hi.width <= a.pitch;
    }
  }
  TORCH_CHECK_VALUE(ok, "out shares memory with ", what);
}
void apart(const Tensor& out, const optional<Tensor>& in, bool exact_ok, const char* what) {
  if (in) apart(out, *in, exact_ok, what);
}

// The [m, n] view of a caller's output.
Tensor out_rows(const Tensor& out, at::IntArrayRef lead, int64_t m, int64_t n,
                at::ScalarType type) {
  auto shape = lead.vec();
  shape.push_back(n);
  TORCH_CHECK_VALUE(out.scalar_type() == type && out.sizes() == at::IntArrayRef(shape),
                    "out must be ", type, " ", at::IntArrayRef(shape));
  TORCH_CHECK_VALUE(out.dim() == 2 ||
                        at::detail::computeStride(out.sizes(), out.strides(), at::DimVector{m, n}),
                    "out must be a view of rows at one stride");
  Tensor o = out.dim() == 2 ? out : out.view({m, n});
  TORCH_CHECK_VALUE(m == 0 || rows_aligned(o), "out must have contiguous, 16-byte aligned rows");
  out.unsafeGetTensorImpl()->bump_version();
  return o;
}

struct Extras {
  Tensor bias, residual;
  const void* b = nullptr;
  const void* r = nullptr;
  int64_t ldr = 0;
  Extras(const optional<Tensor>& bias_in, const optional<Tensor>& res_in, int64_t m, int64_t n,
         at::ScalarType type) {
    if (bias_in) {
      TORCH_CHECK_VALUE(bias_in->scalar_type() == type && bias_in->dim() == 1 &&
                            bias_in->size(0) == n,
                        "bias must be ", type, " [", n, "]");
      bias = *bias_in;
      if (bias.stride(0) != 1 || !aligned(bias.data_ptr()))
        bias = bias.clone(at::MemoryFormat::Contiguous);
      b = bias.data_ptr();
    }
    if (res_in) {
      TORCH_CHECK_VALUE(res_in->scalar_type() == type && res_in->numel() == m * n &&
                            res_in->dim() >= 1 && res_in->size(-1) == n,
                        "residual must be ", type, " with ", m, " rows of ", n);
      residual = rows2d(*res_in);
      r = residual.data_ptr();
      ldr = residual.stride(0);
    }
  }
};

void check_act(int64_t act) {
  TORCH_CHECK_VALUE(act == H3B_ACT_NONE || act == H3B_ACT_GELU_TANH,
                    "the MXFP4 products take ACT_NONE or ACT_GELU_TANH");
}

// ---------------------------------------------------------------- MXFP4
void quantize_into(const Call& c, const Tensor& x2, int64_t k, const Tensor& q, const Tensor& sf) {
  const int64_t m = x2.size(0);
  if (m == 0) return;
  check(h3b_mxfp4_quantize(x2.data_ptr(), dtype_code(x2, true, "mxfp4_quantize"), m, k,
                           x2.stride(0), q.data_ptr(), sf.data_ptr(), c.stream()),
        "h3b_mxfp4_quantize");
}

Tensor quantize_input(const Tensor& x) {
  dtype_code(x, true, "mxfp4_quantize");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 32 == 0,
                    "K must be a positive multiple of 32");
  return rows2d(x);
}

std::tuple<Tensor, Tensor> mxfp4_quantize(const Tensor& x) {
  Call c(x);
  const Tensor x2 = quantize_input(x);
  const int64_t m = x2.size(0), k = x2.size(1);
  Tensor q = new_tensor({m, k / 2}, at::kByte, x), sf = new_tensor({sf_bytes(m, k)}, at::kByte, x);
  quantize_into(c, x2, k, q, sf);
  return {q, sf};
}

void mxfp4_quantize_out(const Tensor& x, Tensor q, Tensor sf) {
  Call c(x);
  c.same(q);
  c.same(sf);
  const Tensor x2 = quantize_input(x);
  check_operand(q, sf, x2.size(0), x2.size(1), "mxfp4_quantize");
  apart(q, x, false, "x");
  apart(sf, x, false, "x");
  apart(sf, q, false, "the codes");
  q.unsafeGetTensorImpl()->bump_version();
  sf.unsafeGetTensorImpl()->bump_version();
  quantize_into(c, x2, x2.size(1), q, sf);
}

void dequantize_into(const Call& c, const Tensor& q, const Tensor& sf, int64_t m, int64_t k,
                     const Tensor& out) {
  if (m == 0) return;
  check(h3b_mxfp4_dequantize(q.data_ptr(), sf.data_ptr(), m, k, out.data_ptr(),
                             dtype_code(out, true, "mxfp4_dequantize"), out.stride(0), c.stream()),
        "h3b_mxfp4_dequantize");
}

Tensor mxfp4_dequantize(const Tensor& q, const Tensor& sf, int64_t m, int64_t k,
                        at::ScalarType dtype) {
  Call c(q);
  c.same(sf);
  check_operand(q, sf, m, k, "mxfp4_dequantize");
  TORCH_CHECK_TYPE(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat,
                   "mxfp4_dequantize gives bf16, fp16 or fp32, not ", dtype);
  Tensor out = new_tensor({m, k}, dtype, q);
  dequantize_into(c, q, sf, m, k, out);
  return out;
}

void mxfp4_dequantize_out(const Tensor& q, const Tensor& sf, int64_t m, int64_t k, Tensor out) {
  Call c(q);
  c.same(sf);
  c.same(out);
  check_operand(q, sf, m, k, "mxfp4_dequantize");
  apart(out, q, false, "the codes");
  apart(out, sf, false, "the scales");
  dequantize_into(c, q, sf, m, k, out_rows(out, {m}, m, k, out.scalar_type()));
}

void gemm_into(const Call& c, const Tensor& qa, const Tensor& sfa, int64_t m, const Tensor& qb,
               const Tensor& sfb, int64_t n, int64_t k, const Extras& e, int64_t act,
               const Tensor& o) {
  if (m == 0) return;
  check(h3b_mxfp4_gemm(qa.data_ptr(), sfa.data_ptr(), m, qb.data_ptr(), sfb.data_ptr(), n, k, e.b,
                       (int)act, e.r, e.ldr, o.data_ptr(), dtype_code(o, false, "mxfp4_gemm"),
                       o.stride(0), c.stream()),
        "h3b_mxfp4_gemm");
}

void gemm_checks(const Call& c, const Tensor& sfa, const Tensor& qa, int64_t m, const Tensor& qb,
                 const Tensor& sfb, int64_t n, int64_t k, const optional<Tensor>& bias,
                 int64_t act, const optional<Tensor>& residual) {
  c.same(sfa);
  c.same(qb);
  c.same(sfb);
  c.same(bias);
  c.same(residual);
  check_n(n);
  check_act(act);
  check_operand(qa, sfa, m, k, "mxfp4_gemm: A");
  check_operand(qb, sfb, n, k, "mxfp4_gemm: B");
}

Tensor mxfp4_gemm(const Tensor& qa, const Tensor& sfa, int64_t m, const Tensor& qb,
                  const Tensor& sfb, int64_t n, int64_t k, const optional<Tensor>& bias,
                  int64_t act, const optional<Tensor>& residual, at::ScalarType dtype) {
  Call c(qa);
  gemm_checks(c, sfa, qa, m, qb, sfb, n, k, bias, act, residual);
  TORCH_CHECK_TYPE(dtype == at::kBFloat16 || dtype == at::kHalf,
                   "mxfp4_gemm gives bf16 or fp16, not ", dtype);
  const Extras e(bias, residual, m, n, dtype);
  Tensor out = new_tensor({m, n}, dtype, qa);
  gemm_into(c, qa, sfa, m, qb, sfb, n, k, e, act, out);
  return out;
}

void mxfp4_gemm_out(const Tensor& qa, const Tensor& sfa, int64_t m, const Tensor& qb,
                    const Tensor& sfb, int64_t n, int64_t k, const optional<Tensor>& bias,
                    int64_t act, const optional<Tensor>& residual, Tensor out) {
  Call c(qa);
  gemm_checks(c, sfa, qa, m, qb, sfb, n, k, bias, act, residual);
  c.same(out);
  dtype_code(out, false, "mxfp4_gemm");
  apart(out, qa, false, "A");
  apart(out, residual, true, "the residual");
  apart(out, bias, false, "the bias");
  const Extras e(bias, residual, m, n, out.scalar_type());
  gemm_into(c, qa, sfa, m, qb, sfb, n, k, e, act, out_rows(out, {m}, m, n, out.scalar_type()));
}

Tensor product_input(const Tensor& x, int64_t k) {
  dtype_code(x, false, "an MXFP4 product");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == k, "activation width ",
                    x.dim() ? x.size(-1) : 0, " != in_features ", k);
  return rows2d(x);
}

void linear_into(const Call& c, const Tensor& x2, const Tensor& qb, const Tensor& sfb, int64_t n,
                 int64_t k, const Extras& e, int64_t act, const Tensor& o, int64_t ldo) {
  const int64_t m = x2.size(0);
  if (m == 0) return;
  const int64_t bytes = h3b_mxfp4_linear_ws(m, n, k);
  const Tensor ws = scratch(bytes, x2);
  check(h3b_mxfp4_linear(x2.data_ptr(), dtype_code(x2, false, "mxfp4_linear"), m, x2.stride(0),
                         qb.data_ptr(), sfb.data_ptr(), n, k, e.b, (int)act, e.r, e.ldr,
                         o.data_ptr(), ldo, ptr(ws), bytes, c.stream()),
        "h3b_mxfp4_linear");
}

void linear_checks(const Call& c, const Tensor& qb, const Tensor& sfb, int64_t n, int64_t k,
                   const optional<Tensor>& bias, int64_t act, const optional<Tensor>& residual) {
  c.same(qb);
  c.same(sfb);
  c.same(bias);
  c.same(residual);
  check_n(n);
  check_act(act);
  check_operand(qb, sfb, n, k, "mxfp4_linear: weight");
}

Tensor mxfp4_linear(const Tensor& x, const Tensor& qb, const Tensor& sfb, int64_t n, int64_t k,
                    const optional<Tensor>& bias, int64_t act, const optional<Tensor>& residual) {
  Call c(x);
  linear_checks(c, qb, sfb, n, k, bias, act, residual);
  const Tensor x2 = product_input(x, k);
  const Extras e(bias, residual, x2.size(0), n, x.scalar_type());
  Tensor out = new_out(x, n, x.scalar_type());
  linear_into(c, x2, qb, sfb, n, k, e, act, out, n);
  return out;
}

void mxfp4_linear_out(const Tensor& x, const Tensor& qb, const Tensor& sfb, int64_t n, int64_t k,
                      const optional<Tensor>& bias, int64_t act, const optional<Tensor>& residual,
                      Tensor out) {
  Call c(x);
  linear_checks(c, qb, sfb, n, k, bias, act, residual);
  c.same(out);
  apart(out, x, false, "x");
  apart(out, residual, true, "the residual");
  apart(out, bias, false, "the bias");
  const Tensor x2 = product_input(x, k);
  const Extras e(bias, residual, x2.size(0), n, x.scalar_type());
  const Tensor o = out_rows(out, x.sizes().slice(0, x.dim() - 1), x2.size(0), n, x.scalar_type());
  linear_into(c, x2, qb, sfb, n, k, e, act, o, o.dim() == 2 ? o.stride(0) : n);
}

void ffn_into(const Call& c, const Tensor& x2, const Tensor& qu, const Tensor& sfu,
              const Tensor& qd, const Tensor& sfd, int64_t n, int64_t f, const Extras& e,
              const Tensor& o, int64_t ldo) {
  const int64_t m = x2.size(0);
  if (m == 0) return;
  const int64_t bytes = h3b_mxfp4_ffn_ws(m, n, f);
  const Tensor ws = scratch(bytes, x2);
  check(h3b_mxfp4_ffn(x2.data_ptr(), dtype_code(x2, false, "mxfp4_ffn"), m, x2.stride(0),
                      qu.data_ptr(), sfu.data_ptr(), qd.data_ptr(), sfd.data_ptr(), n, f, e.r,
                      e.ldr, o.data_ptr(), ldo, ws.data_ptr(), bytes, c.stream()),
        "h3b_mxfp4_ffn");
}

void ffn_checks(const Call& c, const Tensor& qu, const Tensor& sfu, const Tensor& qd,
                const Tensor& sfd, int64_t n, int64_t f, const optional<Tensor>& residual) {
  c.same(qu);
  c.same(sfu);
  c.same(qd);
  c.same(sfd);
  c.same(residual);
  TORCH_CHECK_VALUE(f > 0 && f % 128 == 0, "feed-forward width ", f,
                    " must be a positive multiple of 128");
  check_operand(qu, sfu, 2 * f, n, "mxfp4_ffn: up projection");
  check_operand(qd, sfd, n, f, "mxfp4_ffn: down projection");
}

Tensor mxfp4_ffn(const Tensor& x, const Tensor& qu, const Tensor& sfu, const Tensor& qd,
                 const Tensor& sfd, int64_t n, int64_t f, const optional<Tensor>& residual) {
  Call c(x);
  ffn_checks(c, qu, sfu, qd, sfd, n, f, residual);
  const Tensor x2 = product_input(x, n);
  const Extras e(std::nullopt, residual, x2.size(0), n, x.scalar_type());
  Tensor out = new_out(x, n, x.scalar_type());
  ffn_into(c, x2, qu, sfu, qd, sfd, n, f, e, out, n);
  return out;
}

void mxfp4_ffn_out(const Tensor& x, const Tensor& qu, const Tensor& sfu, const Tensor& qd,
                   const Tensor& sfd, int64_t n, int64_t f, const optional<Tensor>& residual,
                   Tensor out) {
  Call c(x);
  ffn_checks(c, qu, sfu, qd, sfd, n, f, residual);
  c.same(out);
  apart(out, x, true, "x");
  apart(out, residual, true, "the residual");
  const Tensor x2 = product_input(x, n);
  const Extras e(std::nullopt, residual, x2.size(0), n, x.scalar_type());
  const Tensor o = out_rows(out, x.sizes().slice(0, x.dim() - 1), x2.size(0), n, x.scalar_type());
  ffn_into(c, x2, qu, sfu, qd, sfd, n, f, e, o, o.stride(0));
}

// ---------------------------------------------------------------- windowed attention
struct Rule {
  int64_t left, right, sinks;
  bool causal;
  double scale;
};

void check_rule(const Rule& r, int64_t heads, int64_t kv_heads, int64_t d) {
  TORCH_CHECK_VALUE(d == 64 || d == 128, "head_dim must be 64 or 128, not ", d);
  TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, heads,
                    " query heads are not a multiple of ", kv_heads, " key heads");
  TORCH_CHECK_VALUE(r.left >= 0 && r.right >= 0 && r.sinks >= 0,
                    "window sides and sinks must not be negative");
  const float scale = (float)r.scale;              // the kernels', times log2(e)
  TORCH_CHECK_VALUE(scale > 0 && std::isfinite(scale * 1.4426950408889634f),
                    "scale must be positive, and scale * log2(e) finite in fp32");
}

// Row ranges of the documents that boundaries give.
struct Docs {
  std::vector<int32_t> start, len;
  int64_t covered = 0;
  Docs(at::IntArrayRef cu, int64_t rows, const char* what) {
    bool ok = !cu.empty() && cu.front() >= 0 && cu.back() <= rows && rows <= (1 << 30);
    for (size_t i = 0; ok && i + 1 < cu.size(); ++i) ok = cu[i] <= cu[i + 1];
    TORCH_CHECK_VALUE(ok, what, " must rise from 0 or more to at most ", rows);
    start.reserve(cu.size());
    len.reserve(cu.size());
    for (size_t i = 0; i + 1 < cu.size(); ++i) {
      start.push_back((int32_t)cu[i]);
      len.push_back((int32_t)(cu[i + 1] - cu[i]));
      covered += len.back();
    }
  }
};

struct Packed {
  Tensor q, k, v;
  Docs qd, kd;
  static at::IntArrayRef keys(at::IntArrayRef cu, const at::OptionalIntArrayRef& cu_k) {
    return cu_k ? *cu_k : cu;
  }
  Packed(const Call& c, const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t heads,
         int64_t kv_heads, int64_t d, at::IntArrayRef cu, const at::OptionalIntArrayRef& cu_k,
         const Rule& r)
      : q(ready(c, q_)),
        k(ready(c, k_)),
        v(ready(c, v_)),
        qd(cu, q.size(0), "cu_seqlens"),
        kd(keys(cu, cu_k), k.size(0), "cu_seqlens_k") {
    check_rule(r, heads, kv_heads, d);
    dtype_code(q, false, "attention");
    TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                     "q, k, v must be of one type");
    TORCH_CHECK_VALUE(q.size(1) == heads * d && k.sizes() == v.sizes() &&
                          k.size(1) == kv_heads * d,
                      "q must be [rows, heads * head_dim], k and v [rows, kv_heads * head_dim]");
    TORCH_CHECK_VALUE(qd.start.size() == kd.start.size(),
                      "cu_seqlens and cu_seqlens_k name different numbers of documents");
  }
  static Tensor ready(const Call& c, const Tensor& t) {
    c.same(t);
    return rows2d(t);
  }
};

void window_into(const Call& c, const Packed& p, int64_t heads, int64_t kv_heads, int64_t d,
                 const Rule& r, const Tensor& o) {
  if (p.qd.covered == 0) return;
  const int docs = (int)p.qd.start.size();
  const int64_t bytes = h3b_attention_window_ws(p.qd.len.data(), p.kd.len.data(), docs, (int)heads,
                                                (int)d, r.left, r.right, r.sinks);
  const Tensor ws = scratch(bytes, p.q);
  check(h3b_attention_window(p.q.data_ptr(), p.q.size(0), p.q.stride(0), p.k.data_ptr(),
                             p.k.stride(0), p.v.data_ptr(), p.v.stride(0), p.k.size(0),
                             dtype_code(p.q, false, "attention"), (int)heads, (int)kv_heads,
                             (int)d, p.qd.start.data(), p.qd.len.data(), p.kd.start.data(),
                             p.kd.len.data(), docs, r.left, r.right, r.sinks, r.causal,
                             (float)r.scale, o.data_ptr(), o.stride(0),
                             ptr(ws), bytes, c.stream()),
        "h3b_attention_window");
}

Tensor attention_window(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads,
                        int64_t kv_heads, int64_t d, at::IntArrayRef cu,
                        at::OptionalIntArrayRef cu_k, int64_t left, int64_t right, int64_t sinks,
                        bool causal, double scale) {
  Call c(q);
  const Rule r{left, right, sinks, causal, scale};
  const Packed p(c, q, k, v, heads, kv_heads, d, cu, cu_k, r);
  // rows of no document read as zeros
  Tensor out = p.qd.covered == p.q.size(0) ? new_tensor({p.q.size(0), heads * d}, q.scalar_type(), q)
                                           : at::zeros({p.q.size(0), heads * d}, q.options());
  window_into(c, p, heads, kv_heads, d, r, out);
  return out;
}

void attention_window_out(const Tensor& q, const Tensor& k, const Tensor& v, int64_t heads,
                          int64_t kv_heads, int64_t d, at::IntArrayRef cu,
                          at::OptionalIntArrayRef cu_k, int64_t left, int64_t right,
                          int64_t sinks, bool causal, double scale, Tensor out) {
  Call c(q);
  c.same(out);
  const Rule r{left, right, sinks, causal, scale};
  const Packed p(c, q, k, v, heads, kv_heads, d, cu, cu_k, r);
  const int64_t rows = p.q.size(0);
  apart(out, q, true, "q");
  apart(out, k, false, "k");
  apart(out, v, false, "v");
  window_into(c, p, heads, kv_heads, d, r,
              out_rows(out, {rows}, rows, heads * d, q.scalar_type()));
}

bool decode_strides(const Tensor& t) {
  return t.stride(3) == 1 && (t.stride(0) | t.stride(1) | t.stride(2)) % 8 == 0 &&
         aligned(t.data_ptr());
}

void decode_into(const Call& c, const Tensor& q_in, const Tensor& k, const Tensor& v,
                 const Tensor& len, const Rule& r, const Tensor& out) {
  c.same(k);
  c.same(v);
  c.same(len);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes(),
                    "q must be [B, n_new, heads, D], k and v [B, room, kv_heads, D]");
  const int64_t B = q_in.size(0), n = q_in.size(1), heads = q_in.size(2), d = q_in.size(3);
  TORCH_CHECK_VALUE(k.size(0) == B && k.size(3) == d, "q, k and v must agree on batch and head_dim");
  check_rule(r, heads, k.size(2), d);
  const int dt = dtype_code(q_in, false, "attention");
  TORCH_CHECK_TYPE(k.scalar_type() == q_in.scalar_type() && v.scalar_type() == q_in.scalar_type(),
                   "q, k, v must be of one type");
  TORCH_CHECK_VALUE(len.scalar_type() == at::kInt && len.dim() == 1 && len.size(0) == B &&
                        len.is_contiguous(),
                    "kv_len must be a contiguous int32 [", B, "]");
  TORCH_CHECK_VALUE(out.scalar_type() == q_in.scalar_type() && out.sizes() == q_in.sizes() &&
                        out.is_contiguous() && aligned(out.data_ptr()),
                    "out must be a contiguous, 16-byte aligned ", q_in.scalar_type(), " ",
                    q_in.sizes());
  TORCH_CHECK_VALUE(k.numel() == 0 || (decode_strides(k) && decode_strides(v)),
                    "caches need a contiguous head_dim and 16-byte aligned rows");
  if (out.numel() == 0) return;
  TORCH_CHECK_VALUE(B <= 65535 && n <= 65535 &&
                        (n * (heads / k.size(2)) + 15) / 16 * k.size(2) <= 65535,
                    "at most 65535 sequences, and 65535 blocks of 16 rows that share a key head, "
                    "not ", B, " and ", n, " new tokens of ", heads, " heads");
  const Tensor q = decode_strides(q_in) ? q_in : q_in.clone(at::MemoryFormat::Contiguous);
  static const int64_t none[4] = {0, 0, 0, 0};       // an empty cache's strides mean nothing
  const bool empty = k.numel() == 0;
  check(h3b_attention_window_decode(q.data_ptr(), q.strides().data(), k.data_ptr(),
                                    empty ? none : k.strides().data(), v.data_ptr(),
                                    empty ? none : v.strides().data(),
                                    len.const_data_ptr<int32_t>(), B, k.size(1), n, dt, (int)heads,
                                    (int)k.size(2), (int)d, r.left, r.right, r.sinks, r.causal,
                                    (float)r.scale, out.data_ptr(), c.stream()),
        "h3b_attention_window_decode");
}

Tensor attention_window_decode(const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& len, int64_t left, int64_t right, int64_t sinks,
                               bool causal, double scale) {
  Call c(q);
  Tensor out = new_tensor(q.sizes(), q.scalar_type(), q);
  decode_into(c, q, k, v, len, Rule{left, right, sinks, causal, scale}, out);
  return out;
}

void attention_window_decode_out(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& len, int64_t left, int64_t right, int64_t sinks,
                                 bool causal, double scale, Tensor out) {
  Call c(q);
  c.same(out);
  apart(out, q, true, "q");
  apart(out, k, false, "k");
  apart(out, v, false, "v");
  decode_into(c, q, k, v, len, Rule{left, right, sinks, causal, scale}, out);
  out.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

#define MX_GEMM "Tensor qa, Tensor sfa, int m, Tensor qb, Tensor sfb, int n, int k, Tensor? bias, int act, Tensor? residual"
#define MX_LINEAR "Tensor x, Tensor qb, Tensor sfb, int n, int k, Tensor? bias, int act, Tensor? residual"
#define MX_FFN "Tensor x, Tensor qu, Tensor sfu, Tensor qd, Tensor sfd, int n, int f, Tensor? residual"
#define WINDOW "Tensor q, Tensor k, Tensor v, int heads, int kv_heads, int head_dim, int[] cu_seqlens, int[]? cu_seqlens_k, int left, int right, int sinks, bool causal, float scale"
#define DECODE "Tensor q, Tensor k, Tensor v, Tensor kv_len, int left, int right, int sinks, bool causal, float scale"

TORCH_LIBRARY_FRAGMENT(h3b, m) {
  m.def("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("mxfp4_quantize_out(Tensor x, Tensor(a!) q, Tensor(b!) sf) -> ()");
  m.def("mxfp4_dequantize(Tensor q, Tensor sf, int m, int k, ScalarType dtype) -> Tensor");
  m.def("mxfp4_dequantize_out(Tensor q, Tensor sf, int m, int k, Tensor(a!) out) -> ()");
  m.def("mxfp4_gemm(" MX_GEMM ", ScalarType dtype) -> Tensor");
  m.def("mxfp4_gemm_out(" MX_GEMM ", Tensor(a!) out) -> ()");
  m.def("mxfp4_linear(" MX_LINEAR ") -> Tensor");
  m.def("mxfp4_linear_out(" MX_LINEAR ", Tensor(a!) out) -> ()");
  m.def("mxfp4_ffn(" MX_FFN ") -> Tensor");
  m.def("mxfp4_ffn_out(" MX_FFN ", Tensor(a!) out) -> ()");
  m.def("attention_window(" WINDOW ") -> Tensor");
  m.def("attention_window_out(" WINDOW ", Tensor(a!) out) -> ()");
  m.def("attention_window_decode(" DECODE ") -> Tensor");
  m.def("attention_window_decode_out(" DECODE ", Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(h3b, CUDA, m) {
  m.impl("mxfp4_quantize", &mxfp4_quantize);
  m.impl("mxfp4_quantize_out", &mxfp4_quantize_out);
  m.impl("mxfp4_dequantize", &mxfp4_dequantize);
  m.impl("mxfp4_dequantize_out", &mxfp4_dequantize_out);
  m.impl("mxfp4_gemm", &mxfp4_gemm);
  m.impl("mxfp4_gemm_out", &mxfp4_gemm_out);
  m.impl("mxfp4_linear", &mxfp4_linear);
  m.impl("mxfp4_linear_out", &mxfp4_linear_out);
  m.impl("mxfp4_ffn", &mxfp4_ffn);
  m.impl("mxfp4_ffn_out", &mxfp4_ffn_out);
  m.impl("attention_window", &attention_window);
  m.impl("attention_window_out", &attention_window_out);
  m.impl("attention_window_decode", &attention_window_decode);
  m.impl("attention_window_decode_out", &attention_window_decode_out);
}

// Inference only, as the package's other operators: results carry no gradient
// (without this, backward() would run and leave the inputs' gradients out).
TORCH_LIBRARY_IMPL(h3b, Autograd, m) {
  for (const char* name :
       {"mxfp4_quantize", "mxfp4_quantize_out", "mxfp4_dequantize", "mxfp4_dequantize_out",
        "mxfp4_gemm", "mxfp4_gemm_out", "mxfp4_linear", "mxfp4_linear_out", "mxfp4_ffn",
        "mxfp4_ffn_out", "attention_window", "attention_window_out", "attention_window_decode",
        "attention_window_decode_out"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}
