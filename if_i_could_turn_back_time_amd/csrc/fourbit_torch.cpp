// torch's way in.  The packed linear layer's call path from torch: one native call per forward (and per activation
// gradient) instead of a dozen Python, ctypes and dispatcher steps.  It launches the kernels that
// linear.py's packed_linear launches, on x converted as there, and takes workspaces from the
// allocator; what it does not recognise (another dtype, a refused shape, a wrapped tensor or one
// with a forward-mode tangent, a bias that is no vector, an active dispatch mode) it leaves to
// packed_linear by returning None.  A decode call of a 4096^2 layer takes 5 us on the GPU and took
// 22 us of host time through Python.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <stdexcept>

#include "fourbit.h"

namespace py = pybind11;

namespace {

constexpr int64_t kMaxGemvBatch = 16;
constexpr int64_t kMaxGemmK = 1 << 22;  // fb_gemm's limits
constexpr int64_t kMaxGemmRows = 1 << 24;
constexpr int64_t kMaxRotatedValues = 1 << 29;  // of x, rotated at once: a copy of 1 GiB
// Rows of grad_y at once: bounds fb_grad_x's 16-bit terms of them, and each pass's decode of W
// is under 1% of its products.
constexpr int64_t kGradRows = 8192;
constexpr int64_t kGradVocab = 1 << 18;  // fb_grad_x's limit of a weight's rows

void check(int code) {
  if (code != FB_OK) throw std::runtime_error(fb_strerror(code));
}

int dtype_code(at::ScalarType t) {
  return t == at::kHalf ? FB_DT_F16 : t == at::kBFloat16 ? FB_DT_BF16 : t == at::kFloat ? FB_DT_F32 : -1;
}

// A plain dense GPU tensor whose memory this code may read: no functorch wrapper, fake or
// functional tensor, and no forward-mode tangent, which only torch operations carry on.
bool plain(const at::Tensor& t) {
  const auto ks = t.key_set();
  return !t._fw_grad(0).defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() &&
         !ks.has(c10::DispatchKey::Python) && !ks.has(c10::DispatchKey::Functionalize) &&
         !ks.has(c10::DispatchKey::FuncTorchBatched) &&
         !ks.has(c10::DispatchKey::FuncTorchGradWrapper) && !t.is_neg() && !t.is_conj();
}

// Whether somebody watches the operators.
bool watched() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer) ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

void* ptr_or_null(const at::Tensor& t, size_t bytes) { return bytes ? t.data_ptr() : nullptr; }

// F.linear(x, W, bias) for a packed W, no gradients; None where packed_linear has to decide.
std::optional<at::Tensor> linear_forward(const at::Tensor& x, const at::Tensor& wdev, int64_t N,
                                         int64_t K, int64_t fmt, int64_t fwht_block, bool f16_exact,
                                         bool fp4_mfma, const std::optional<at::Tensor>& bias,
                                         bool bf16_exact) {
  if (watched() || !plain(x) || !plain(wdev) || x.device() != wdev.device() || x.dim() < 1 ||
      x.size(-1) != K || K < 1 || x.numel() == 0)
    return std::nullopt;
  // a bias of more dimensions broadcasts against the [M, N] product, not against y's shape
  if (bias && (!plain(*bias) || bias->device() != x.device() || bias->dim() > 1))
    return std::nullopt;
  const int xdt = dtype_code(x.scalar_type());
  if (xdt < 0) return std::nullopt;
  const bool e2m1 = fmt == FB_FMT_E2M1;
  if (fp4_mfma && (!e2m1 || fwht_block)) return std::nullopt;
  int kdt = xdt;  // the kernels' activation dtype
  if (!e2m1 || fwht_block)
    kdt = FB_DT_F16;
  else if (fp4_mfma || xdt == FB_DT_F32)
    kdt = FB_DT_BF16;
  if (e2m1 && kdt == FB_DT_F16 && !f16_exact) return std::nullopt;
  const int64_t kp = (K + 127) / 128 * 128, M = x.numel() / K;
  if (M > INT32_MAX || (M > kMaxGemvBatch && kp > kMaxGemmK)) return std::nullopt;
  // the GEMM decodes to bf16; the split of more than one GEMV batch is linear.py's
  if (M > kMaxGemvBatch && fp4_mfma && !bf16_exact) return std::nullopt;

  fb_shape_t s{};
  s.N = (int32_t)N;
  s.K = (int32_t)kp;
  s.B = (int32_t)std::min(M, fwht_block ? std::min(kMaxGemmRows, kMaxRotatedValues / kp / 16 * 16)
                                       : kMaxGemmRows);  // rows of a call
  s.group = e2m1 ? 32 : 128;
  s.fmt = (int32_t)fmt;
  s.fwht_block = (int32_t)fwht_block;
  s.x_dtype = kdt;
  s.y_dtype = xdt;
  if ((size_t)wdev.numel() < fb_device_bytes(&s) || !fb_device_bytes(&s)) return std::nullopt;

  c10::DeviceGuard guard(x.device());
  void* const stream = stream_of(x);
  const at::Tensor xc = x.is_contiguous() ? x : x.contiguous();
  at::Tensor xk = xc;
  if (kdt != xdt || kp != K) {
    xk = at::empty({M, kp}, x.options().dtype(kdt == FB_DT_F16 ? at::kHalf : at::kBFloat16));
    check(fb_cast_rows(xc.data_ptr(), xdt, (int32_t)M, (int32_t)K, xk.data_ptr(), kdt,
                       (int32_t)kp, stream));
  }
  if (reinterpret_cast<uintptr_t>(xk.data_ptr()) & 15u) return std::nullopt;
  // a bias that is a plain vector is added by the GEMM, or by one small kernel
  const bool vector_bias = bias && bias->dim() == 1 && bias->size(0) == N &&
                           bias->is_contiguous() && dtype_code(bias->scalar_type()) >= 0;
  const int bdt = vector_bias ? dtype_code(bias->scalar_type()) : 0;
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  at::Tensor y = at::empty(sizes, x.options());
  if (M > kMaxGemvBatch) {
    const int64_t step = s.B;
    for (int64_t r = 0; r < M; r += step) {
      s.B = (int32_t)std::min(step, M - r);
      const size_t need = fb_gemm_workspace_bytes(&s);
      const at::Tensor ws = need ? scratch(need, x) : at::Tensor();
      check(fb_gemm(wdev.data_ptr(), static_cast<const char*>(xk.data_ptr()) + r * kp * 2,
                    static_cast<char*>(y.data_ptr()) + r * N * y.element_size(), &s,
                    vector_bias ? bias->data_ptr() : nullptr, bdt, ptr_or_null(ws, need), need,
                    stream));
    }
    if (vector_bias) return y;
  } else if (fp4_mfma) {
    const size_t need = fb_mx_workspace_bytes(&s);
    if (!need) return std::nullopt;
    const at::Tensor ws = scratch(need, x);
    check(fb_gemv_mx(wdev.data_ptr(), xk.data_ptr(), y.data_ptr(), &s, ws.data_ptr(), need,
                     stream));
  } else {
    const size_t need = fb_workspace_bytes(&s);
    const at::Tensor ws = need ? scratch(need, x) : at::Tensor();
    check(fb_gemv(wdev.data_ptr(), xk.data_ptr(), y.data_ptr(), &s, ptr_or_null(ws, need), need,
                  stream));
  }
  if (vector_bias)
    check(fb_add_bias(y.data_ptr(), xdt, (int32_t)M, (int32_t)N, bias->data_ptr(), bdt, stream));
  else if (bias)
    y.add_(bias->scalar_type() == y.scalar_type() ? *bias : bias->to(y.scalar_type()));
  return y;
}

// gx[M, K] = (gy . W) H for gy [M, N], in xdtype; None where the caller has to decide.
std::optional<at::Tensor> linear_grad_x(const at::Tensor& gy, const at::Tensor& wdev, int64_t N,
                                        int64_t K, int64_t fmt, int64_t fwht_block, bool f16_exact,
                                        at::ScalarType xt) {
  const int gdt = dtype_code(gy.scalar_type()), xdt = dtype_code(xt);
  const int64_t kp = (K + 127) / 128 * 128;
  if (watched() || !plain(gy) || !plain(wdev) || gy.device() != wdev.device() || gy.dim() != 2 ||
      gy.size(1) != N || gdt < 0 || xdt < 0 || gy.numel() == 0)
    return std::nullopt;
  fb_shape_t s{};
  s.N = (int32_t)N;
  s.K = (int32_t)kp;
  s.B = (int32_t)std::min(gy.size(0), kGradRows);
  s.group = fmt == FB_FMT_E2M1 ? 32 : 128;
  s.fmt = (int32_t)fmt;
  s.fwht_block = (int32_t)fwht_block;
  s.x_dtype = FB_DT_F16;
  s.y_dtype = gdt;
  if (!fb_grad_x_workspace_bytes(&s, f16_exact) || (size_t)wdev.numel() < fb_device_bytes(&s))
    return std::nullopt;
  c10::DeviceGuard guard(gy.device());
  const at::Tensor g = gy.contiguous();
  at::Tensor gx = at::empty({gy.size(0), kp}, gy.options().dtype(xt));
  for (int64_t r = 0; r < gy.size(0); r += kGradRows) {
    s.B = (int32_t)std::min(gy.size(0) - r, kGradRows);
    const size_t need = fb_grad_x_workspace_bytes(&s, f16_exact);
    const at::Tensor ws = scratch(need, gy);
    check(fb_grad_x(wdev.data_ptr(), static_cast<const char*>(g.data_ptr()) + r * N * g.element_size(),
                    static_cast<char*>(gx.data_ptr()) + r * kp * gx.element_size(), &s, xdt,
                    f16_exact, ws.data_ptr(), need, stream_of(gy)));
  }
  return kp == K ? gx : gx.narrow(1, 0, K).contiguous();
}

// The bias gradient: gy's column sums in bdtype; None where the caller has to decide.
std::optional<at::Tensor> linear_grad_bias(const at::Tensor& gy, at::ScalarType bt) {
  const int gdt = dtype_code(gy.scalar_type()), bdt = dtype_code(bt);
  if (watched() || !plain(gy) || gy.dim() != 2 || gdt < 0 || bdt < 0 || gy.numel() == 0 ||
      gy.size(0) > INT32_MAX || gy.size(1) > INT32_MAX)
    return std::nullopt;
  c10::DeviceGuard guard(gy.device());
  const at::Tensor g = gy.contiguous();
  at::Tensor gb = at::empty({gy.size(1)}, gy.options().dtype(bt));
  const int32_t M = (int32_t)gy.size(0), N = (int32_t)gy.size(1);
  const size_t need = fb_grad_bias_workspace_bytes(M, N);
  const at::Tensor ws = need ? scratch(need, gy) : at::Tensor();
  check(fb_grad_bias_ws(g.data_ptr(), gdt, M, N, gb.data_ptr(), bdt, ptr_or_null(ws, need), need,
                        stream_of(gy)));
  return gb;
}

// y, which holds bias [N] already, as a function of it.  A node of its own, and one that knows
// which gradients a backward pass asks for: autograd runs a Python function's whole backward for
// any one of its inputs, so as an input of linear.py's _PackedLinearFn the bias's gradient alone
// would compute gx too.
struct AddedBias : torch::autograd::Function<AddedBias> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& y,
                            const at::Tensor& bias) {
    ctx->mark_dirty({y});
    ctx->saved_data["dtype"] = bias.scalar_type();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const at::Tensor& gy = grads[0];
    at::Tensor gb;
    if (ctx->needs_input_grad(1)) {
      const at::ScalarType bt = ctx->saved_data["dtype"].toScalarType();
      std::optional<at::Tensor> sums;
      if (!at::GradMode::is_enabled()) sums = linear_grad_bias(gy, bt);
      gb = sums ? *sums : gy.sum(0).to(bt);
    }
    return {gy, gb};
  }
};

at::Tensor added_bias(const at::Tensor& y, const at::Tensor& bias) {
  return AddedBias::apply(y, bias);
}

// ---------------------------------------------------------------------------------
// The 8-bit key/value cache and the token log probabilities: what kvcache.py and logprobs.py
// call.  There is no other path, so what does not fit is refused here, by name.
// ---------------------------------------------------------------------------------
void want(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

void want_plain(const at::Tensor& t, const at::Tensor& like, const char* what) {
  want(t.defined() && plain(t), what);
  want(t.device() == like.device(), "all tensors must be on one GPU");
}

void no_grad_through(std::initializer_list<at::Tensor> ts, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor& t : ts)
    if (t.requires_grad()) throw std::runtime_error(what);
}

// What these calls write in place raises its version, as torch's own operators do, so that a graph
// that saved it notices.
void written(std::initializer_list<at::Tensor> ts) {
  for (const at::Tensor& t : ts)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A trace, or a mode that records or replaces torch's operators, would hold the results as constants
// or buffers that nobody fills.
void not_recorded() {
  using Key = c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer) ||
      Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FUNCTIONAL))
    throw std::runtime_error("this call is no torch operator: it cannot be traced or recorded (a HIP "
                             "graph can capture it)");
}

fb_cache_t cache_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks,
                    const at::Tensor& vs) {
  want_plain(k, k, "cache: tensors on a ROCm GPU are needed");
  want_plain(v, k, "cache: tensors on a ROCm GPU are needed");
  want_plain(ks, k, "cache: tensors on a ROCm GPU are needed");
  want_plain(vs, k, "cache: tensors on a ROCm GPU are needed");
  want(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn &&
           ks.scalar_type() == at::kByte && vs.scalar_type() == at::kByte,
       "cache: k and v must be float8_e4m3fn, the scales uint8");
  want(k.dim() == 4 && v.dim() == 5 && ks.dim() == 3 && vs.dim() == 3,
       "cache: k is [pages, heads, page, D], v [pages, heads, page / 16, D, 16], the scales "
       "[pages, heads, page / 32]");
  const int64_t pages = k.size(0), H = k.size(1), P = k.size(2), D = k.size(3);
  want(P % 32 == 0 && v.sizes() == at::IntArrayRef({pages, H, P / 16, D, 16}) &&
           ks.sizes() == at::IntArrayRef({pages, H, P / 32}) && vs.sizes() == ks.sizes(),
       "cache: k is [pages, heads, page, D], v [pages, heads, page / 16, D, 16], the scales "
       "[pages, heads, page / 32], page a multiple of 32");
  want(k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(),
       "cache: tensors must be contiguous");
  want(pages <= INT32_MAX && H <= INT32_MAX && P <= INT32_MAX && D <= INT32_MAX,
       "cache: too large");
  fb_cache_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_scale = static_cast<uint8_t*>(ks.data_ptr());
  c.v_scale = static_cast<uint8_t*>(vs.data_ptr());
  c.pages = pages;
  c.heads = (int32_t)H;
  c.head_dim = (int32_t)D;
  c.page = (int32_t)P;
  return c;
}

// `tokens` rows of x (or q) for the sequences of `table`; what is not given is the most it can be.
fb_seqs_t seqs_of(const at::Tensor& table, const at::Tensor& lens,
                  const std::optional<at::Tensor>& cu, int64_t tokens,
                  std::optional<int64_t> max_new, std::optional<int64_t> max_len, int64_t page,
                  const at::Tensor& like) {
  want_plain(table, like, "table must be a tensor on the cache's GPU");
  want_plain(lens, like, "lens must be a tensor on the cache's GPU");
  want(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) >= 1 &&
           table.size(1) >= 1 && (table.size(1) == 1 || table.stride(1) == 1) &&
           (table.size(0) == 1 || table.stride(0) >= table.size(1)),
       "table must be int32 [sequences, pages] with rows of their own");
  const int64_t B = table.size(0);
  want(B <= 65535 && table.size(1) <= INT32_MAX && tokens <= INT32_MAX,
       "too many sequences, pages or tokens");
  want(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == B &&
           lens.is_contiguous(),
       "the lengths must be int32 [sequences], contiguous");
  if (cu) {
    want_plain(*cu, like, "cu_seqlens must be a tensor on the cache's GPU");
    want(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) == B + 1 &&
             cu->is_contiguous(),
         "cu_seqlens must be int32 [sequences + 1], contiguous");
  } else {
    want(tokens == B, "without cu_seqlens there is one new token a sequence");
  }
  const int64_t capacity = std::min<int64_t>(table.size(1) * page, INT32_MAX);
  want(!max_new || *max_new >= 0, "max_new must not be negative");
  want(!max_len || *max_len >= 0, "max_len must not be negative");
  fb_seqs_t s{};
  s.table = static_cast<const int32_t*>(table.data_ptr());
  s.table_stride = B == 1 ? table.size(1) : table.stride(0);
  s.lens = static_cast<const int32_t*>(lens.data_ptr());
  s.cu = cu ? static_cast<const int32_t*>(cu->data_ptr()) : nullptr;
  s.seqs = (int32_t)B;
  s.max_pages = (int32_t)table.size(1);
  s.tokens = (int32_t)tokens;
  s.max_new = (int32_t)(cu ? std::min(max_new.value_or(tokens), tokens) : 1);
  s.max_len = (int32_t)std::min(max_len.value_or(capacity), capacity);
  return s;
}

// [tokens, heads, D] with any strides between tokens and heads.
void want_rows(const at::Tensor& x, int64_t heads, int64_t D, const char* what) {
  want(x.dim() == 3 && x.size(1) == heads && x.size(2) == D && (x.stride(2) == 1 || D == 1),
       what);
}

// Whether the contiguous rows of a 3-D tensor lie apart, in either order of the other dimensions.
bool rows_apart(const at::Tensor& t) {
  const int64_t n[2] = {t.size(0), t.size(1)}, s[2] = {t.stride(0), t.stride(1)}, w = t.size(2);
  for (int in = 0; in < 2; ++in) {
    const int64_t span = n[in] > 1 ? (n[in] - 1) * s[in] + w : w;
    if ((n[in] <= 1 || s[in] >= w) && (n[1 - in] <= 1 || s[1 - in] >= span)) return true;
  }
  return false;
}

void cache_append(const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
                  const at::Tensor& cvs, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& table, const at::Tensor& start,
                  const std::optional<at::Tensor>& cu, std::optional<int64_t> max_new) {
  not_recorded();
  const fb_cache_t c = cache_of(ck, cv, cks, cvs);
  want_plain(k, ck, "k and v must be tensors on the cache's GPU");
  want_plain(v, ck, "k and v must be tensors on the cache's GPU");
  no_grad_through({k, v}, "the cache carries no gradient: append under torch.no_grad() or "
                          "detached keys and values");
  want_rows(k, c.heads, c.head_dim, "k must be [tokens, heads, D] of the cache, D contiguous");
  want_rows(v, c.heads, c.head_dim, "v must be [tokens, heads, D] of the cache, D contiguous");
  want(k.size(0) == v.size(0) && k.scalar_type() == v.scalar_type(),
       "k and v must agree in tokens and dtype");
  const int dt = dtype_code(k.scalar_type());
  want(dt >= 0, "k and v must be float16, bfloat16 or float32");
  const fb_seqs_t s =
      seqs_of(table, start, cu, k.size(0), max_new, std::nullopt, c.page, ck);
  c10::DeviceGuard guard(ck.device());
  check(fb_cache_append(&c, &s, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                        v.stride(1), dt, stream_of(ck)));
  written({ck, cv, cks, cvs});
}

std::tuple<at::Tensor, std::optional<at::Tensor>> cache_attention(
    const at::Tensor& given, const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks,
    const at::Tensor& cvs, const at::Tensor& table, const at::Tensor& lens,
    const std::optional<at::Tensor>& cu, std::optional<int64_t> max_new,
    std::optional<int64_t> max_len, std::optional<double> scale,
    const std::optional<at::Tensor>& weights, bool want_lse) {
  not_recorded();
  const fb_cache_t c = cache_of(ck, cv, cks, cvs);
  want_plain(given, ck, "q must be a tensor on the cache's GPU");
  no_grad_through({given}, "attention over the cache has no gradient: call it under torch.no_grad() "
                       "or with a detached q");
  want(given.dim() == 3 && given.size(2) == c.head_dim &&
           (given.stride(2) == 1 || c.head_dim == 1),
       "q must be [tokens, query heads, D] with the cache's D, D contiguous");
  want(given.size(1) >= c.heads && given.size(1) % c.heads == 0 && given.size(1) <= INT32_MAX,
       "the query heads must be a multiple of the cache's heads");
  want(given.scalar_type() == at::kHalf || given.scalar_type() == at::kBFloat16,
       "q must be float16 or bfloat16");
  want(!scale || (*scale > 0 && *scale < 1e30), "scale must be positive");
  const fb_seqs_t s = seqs_of(table, lens, cu, given.size(0), max_new, max_len, c.page, ck);
  float* wp = nullptr;
  if (weights) {
    want_plain(*weights, ck, "weights must be a tensor on the cache's GPU");
    want(weights->scalar_type() == at::kFloat && weights->dim() == 3 &&
             weights->size(0) == s.seqs && weights->size(1) == c.heads &&
             weights->size(2) >= std::max(1, s.max_len) && weights->size(2) <= INT32_MAX &&
             weights->stride(2) == 1,
         "weights must be float32 [sequences, heads, at least max_len tokens], the tokens "
         "contiguous");
    want(rows_apart(*weights), "weights must not overlap itself");
    no_grad_through({*weights}, "weights must not require a gradient");
    wp = static_cast<float*>(weights->data_ptr());
  }
  c10::DeviceGuard guard(ck.device());
  // many rows' weights want q 16-byte aligned; a tensor of its own is
  const at::Tensor q = wp && ((reinterpret_cast<uintptr_t>(given.data_ptr()) |
                               (uintptr_t)(given.stride(0) * 2) | (uintptr_t)(given.stride(1) * 2)) &
                              15u)
                           ? given.clone(at::MemoryFormat::Contiguous)
                           : given;
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor lse;
  if (want_lse || wp) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  const size_t need = fb_cache_attention_workspace_bytes(
      &c, &s, (int32_t)q.size(1), wp ? (int32_t)weights->size(2) : 0);
  const at::Tensor ws = need ? scratch(need, q) : at::Tensor();
  check(fb_cache_attention(
      &c, &s, q.data_ptr(), q.stride(0), q.stride(1), (int32_t)q.size(1),
      dtype_code(q.scalar_type()), (float)scale.value_or(1.0 / std::sqrt((double)c.head_dim)),
      out.data_ptr(), lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr, wp,
      wp ? weights->stride(0) : 0, wp ? weights->stride(1) : 0,
      wp ? (int32_t)weights->size(2) : 0, ptr_or_null(ws, need), need, stream_of(ck)));
  if (wp) written({*weights});
  return {out, want_lse ? std::optional<at::Tensor>(lse) : std::nullopt};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> cache_evict(
    const at::Tensor& ck, const at::Tensor& cv, const at::Tensor& cks, const at::Tensor& cvs,
    const at::Tensor& table, const at::Tensor& lens, const at::Tensor& weights, int64_t keep,
    int64_t recent, const at::Tensor& new_table, std::optional<int64_t> max_len) {
  not_recorded();
  const fb_cache_t c = cache_of(ck, cv, cks, cvs);
  want(weights.dim() == 3, "weights must be float32 [sequences, heads, tokens]");
  const fb_seqs_t s = seqs_of(table, lens, std::nullopt, table.size(0), std::nullopt,
                              max_len ? max_len : weights.size(2), c.page, ck);
  want(keep >= 1 && recent >= 0 && recent <= keep && keep <= INT32_MAX,
       "keep must be at least 1, recent between 0 and keep");
  want_plain(weights, ck, "weights must be a tensor on the cache's GPU");
  want(weights.scalar_type() == at::kFloat && weights.dim() == 3 && weights.size(0) == s.seqs &&
           weights.size(1) == c.heads && weights.size(2) >= std::max(1, s.max_len) &&
           weights.size(2) <= INT32_MAX && weights.stride(2) == 1,
       "weights must be float32 [sequences, heads, at least max_len tokens], the tokens "
       "contiguous");
  want_plain(new_table, ck, "new_table must be a tensor on the cache's GPU");
  want(new_table.scalar_type() == at::kInt && new_table.dim() == 2 &&
           new_table.size(0) == s.seqs && new_table.size(1) <= INT32_MAX &&
           new_table.size(1) * c.page >= keep &&
           (new_table.size(1) == 1 || new_table.stride(1) == 1) &&
           (s.seqs == 1 || new_table.stride(0) >= new_table.size(1)),
       "new_table must be int32 [sequences, pages] with pages for keep tokens");
  c10::DeviceGuard guard(ck.device());
  const auto like = weights.options();
  at::Tensor kept = at::empty({s.seqs, c.heads, keep}, like.dtype(at::kInt));
  at::Tensor nw = at::empty({s.seqs, c.heads, keep}, like);
  at::Tensor nl = at::empty({s.seqs}, like.dtype(at::kInt));
  check(fb_cache_evict(&c, &s, static_cast<const float*>(weights.data_ptr()), weights.stride(0),
                       weights.stride(1), (int32_t)weights.size(2), (int32_t)keep,
                       (int32_t)recent, static_cast<const int32_t*>(new_table.data_ptr()),
                       s.seqs == 1 ? new_table.size(1) : new_table.stride(0),
                       (int32_t)new_table.size(1), static_cast<int32_t*>(kept.data_ptr()),
                       static_cast<float*>(nw.data_ptr()), static_cast<int32_t*>(nl.data_ptr()),
                       stream_of(ck)));
  written({ck, cv, cks, cvs});
  return {kept, nl, nw};
}

// logprob, entropy, top_logprobs, top_ids, stats of 2-D logits.
std::vector<at::Tensor> logprobs_forward(const at::Tensor& x, const at::Tensor& token, int64_t top,
                                         bool stats) {
  const int64_t M = x.size(0), V = x.size(1);
  c10::DeviceGuard guard(x.device());
  const auto f = x.options().dtype(at::kFloat);
  at::Tensor lp = at::empty({M}, f), ent = at::empty({M}, f), tl = at::empty({M, top}, f);
  at::Tensor ti = at::empty({M, top}, x.options().dtype(at::kLong));
  at::Tensor st = stats ? at::empty({M, 3}, f) : at::Tensor();
  check(fb_token_logprobs(x.data_ptr(), dtype_code(x.scalar_type()), x.stride(0), M, (int32_t)V,
                          static_cast<const int64_t*>(token.data_ptr()), (int32_t)top,
                          static_cast<float*>(lp.data_ptr()), static_cast<float*>(ent.data_ptr()),
                          top ? static_cast<float*>(tl.data_ptr()) : nullptr,
                          top ? static_cast<int64_t*>(ti.data_ptr()) : nullptr,
                          stats ? static_cast<float*>(st.data_ptr()) : nullptr, stream_of(x)));
  return {lp, ent, tl, ti, st};
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& x, const at::Tensor& token,
                                                int64_t top) {
    const auto r = logprobs_forward(x, token, top, true);
    ctx->save_for_backward({x, token, r[3], r[4], r[1]});
    ctx->mark_non_differentiable({r[3]});
    ctx->set_materialize_grads(false);
    return {r[0], r[1], r[2], r[3]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("token_logprobs has no second derivative");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &token = saved[1], &ids = saved[2], &st = saved[3],
                     &ent = saved[4];
    const int64_t top = ids.size(1);
    c10::DeviceGuard guard(x.device());
    at::Tensor g[3];
    for (int i = 0; i < 3; ++i)
      if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
    const auto ptr = [](const at::Tensor& t) {
      return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr;
    };
    at::Tensor gx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    check(fb_token_logprobs_grad(
        x.data_ptr(), dtype_code(x.scalar_type()), x.stride(0), x.size(0), (int32_t)x.size(1),
        static_cast<const int64_t*>(token.data_ptr()), (int32_t)top,
        static_cast<const int64_t*>(ids.data_ptr()), ptr(st), ptr(ent), ptr(g[0]), ptr(g[1]),
        top ? ptr(g[2]) : nullptr, gx.data_ptr(), stream_of(x)));
    return {gx, at::Tensor(), at::Tensor()};
  }
};

std::vector<at::Tensor> token_logprobs(const at::Tensor& logits, const at::Tensor& tokens,
                                       int64_t top) {
  not_recorded();
  want(logits.defined() && plain(logits), "logits must be a tensor on a ROCm GPU");
  want_plain(tokens, logits, "tokens must be a tensor on the logits' GPU");
  want(dtype_code(logits.scalar_type()) >= 0, "logits must be float16, bfloat16 or float32");
  want(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
       "tokens must be int64 or int32");
  want(logits.dim() >= 1 && tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
       "tokens must have the logits' shape without the last dimension");
  const int64_t V = logits.size(-1);
  want(V >= 1 && V <= (1 << 30), "the last dimension of logits must be the vocabulary");
  want(top >= 0 && top <= FB_LOGPROBS_TOP_MAX && top <= V,
       "top must be between 0 and 64, and at most the vocabulary");
  at::Tensor x = logits;
  if (x.dim() != 2 || (x.stride(1) != 1 && V > 1) || x.stride(0) < 0) x = x.reshape({-1, V});
  if (x.stride(1) != 1 && V > 1) x = x.contiguous();
  const at::Tensor t = tokens.reshape({-1}).to(at::kLong).contiguous();
  std::vector<at::Tensor> r;
  if (at::GradMode::is_enabled() && x.requires_grad())
    r = TokenLogprobs::apply(x, t, top);
  else
    r = logprobs_forward(x, t, top, false);
  r.resize(4);
  if (logits.dim() != 2) {
    auto lead = tokens.sizes().vec();
    r[0] = r[0].view(lead);
    r[1] = r[1].view(lead);
    lead.push_back(top);
    r[2] = r[2].view(lead);
    r[3] = r[3].view(lead);
  }
  return r;
}

// ---------------------------------------------------------------------------------
// Embedding, the seam between blocks, and log probabilities under a head: what embedding.py,
// residual.py and logprobs.py call.
// ---------------------------------------------------------------------------------
void first_derivative(const char* what) {
  if (at::GradMode::is_enabled()) throw std::runtime_error(what);
}

// Autograd hands a gradient to an input's node on the stream that the node was made on.  Of a graph that
// was recorded on another stream and is still alive, that leads out of a capture, which torch ends the
// process for: refused while it can be.
void capturable(std::initializer_list<std::optional<at::Tensor>> inputs) {
  for (const auto& t : inputs) {
    if (!t || !t->defined() || !t->requires_grad()) continue;
    const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream(t->device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(now.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone)
      return;
    const std::shared_ptr<torch::autograd::Node> node =
        t->grad_fn() ? t->grad_fn() : torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto made = node ? node->stream() : std::nullopt;
    if (made && made->id() != now.id())  // (autograd's streams are of another device type by name)
      throw std::runtime_error("an autograd graph of this input recorded outside this capture is still "
                               "alive: drop its results before capturing a backward pass");
  }
}

// x as [rows, width], the values of a row side by side and rows a whole stride apart: a view where
// that can be, else a copy.
at::Tensor as_rows(const at::Tensor& x) {
  at::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < 0)) r = r.contiguous();
  return r;
}
int64_t row_stride(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// tokens as contiguous int64 [rows].
at::Tensor flat_tokens(const at::Tensor& tokens) {
  return tokens.reshape({-1}).to(at::kLong).contiguous();
}
void want_tokens(const at::Tensor& tokens, const at::Tensor& like) {
  want_plain(tokens, like, "tokens must be a tensor on the weight's GPU");
  want(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt,
       "tokens must be int64 or int32");
}

// The shape that is the caller's is given to results where they are made: a view of one that is
// differentiated would be a node of its own.
at::Tensor embedding_forward(const at::Tensor& weight, const at::Tensor& token, at::IntArrayRef sizes,
                             double scale) {
  c10::DeviceGuard guard(weight.device());
  const at::Tensor w = as_rows(weight);
  at::Tensor out = at::empty(sizes, w.options().memory_format(at::MemoryFormat::Contiguous));
  check(fb_embed(w.data_ptr(), row_stride(w), dtype_code(w.scalar_type()), (int32_t)w.size(0),
                 (int32_t)w.size(1), static_cast<const int64_t*>(token.data_ptr()), token.size(0),
                 (float)scale, out.data_ptr(), stream_of(w)));
  return out;
}

struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& w,
                            const at::Tensor& token, const std::vector<int64_t>& sizes, double scale) {
    ctx->save_for_backward({token});
    ctx->saved_data["vocab"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    return embedding_forward(w, token, sizes, scale);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_derivative("token_embedding has no second derivative");
    const at::Tensor token = ctx->get_saved_variables()[0];
    const at::Tensor g = as_rows(grads[0]);
    const int64_t V = ctx->saved_data["vocab"].toInt(), K = g.size(1), M = g.size(0);
    c10::DeviceGuard guard(g.device());
    at::Tensor gw = at::empty({V, K}, g.options().memory_format(at::MemoryFormat::Contiguous));
    const size_t need = fb_embed_grad_workspace_bytes(M, (int32_t)V, (int32_t)K);
    const at::Tensor ws = need ? scratch(need, g) : at::Tensor();
    check(fb_embed_grad(g.data_ptr(), row_stride(g), dtype_code(g.scalar_type()), (int32_t)V,
                        (int32_t)K, static_cast<const int64_t*>(token.data_ptr()), M,
                        (float)ctx->saved_data["scale"].toDouble(), gw.data_ptr(),
                        ptr_or_null(ws, need), need, stream_of(g)));
    return {gw, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor token_embedding(const at::Tensor& tokens, const at::Tensor& weight, double scale) {
  not_recorded();
  want(weight.defined() && plain(weight), "weight must be a tensor on a ROCm GPU");
  want_tokens(tokens, weight);
  want(dtype_code(weight.scalar_type()) >= 0, "weight must be float16, bfloat16 or float32");
  want(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(1) >= 1 &&
           weight.size(0) <= (1 << 30) && weight.size(1) <= (1 << 20),
       "weight must be [vocab, width], a width of at most 2^20");
  want(std::isfinite(scale), "scale must be finite");
  want(tokens.numel() <= (1 << 30), "too many tokens");
  const at::Tensor t = flat_tokens(tokens);
  auto sizes = tokens.sizes().vec();
  sizes.push_back(weight.size(1));
  if (at::GradMode::is_enabled()) capturable({weight});
  return at::GradMode::is_enabled() && weight.requires_grad()
             ? TokenEmbedding::apply(weight, t, sizes, scale)
             : embedding_forward(weight, t, sizes, scale);
}

fb_norm_t norm_of(const at::Tensor& x, const at::Tensor& branch, const at::Tensor& gate,
                  const at::Tensor& weight, const at::Tensor& branch_weight, int64_t gate_rows,
                  double scale, double eps) {
  fb_norm_t n{};
  n.x = x.data_ptr();
  n.x_stride = row_stride(x);
  n.rows = x.size(0);
  n.width = (int32_t)x.size(1);
  n.dtype = dtype_code(x.scalar_type());
  n.weight = weight.data_ptr();
  n.weight_dtype = dtype_code(weight.scalar_type());
  if (branch.defined()) {
    n.branch = branch.data_ptr();
    n.branch_stride = row_stride(branch);
  }
  if (gate.defined()) {
    n.gate = gate.data_ptr();
    n.gate_dtype = dtype_code(gate.scalar_type());
    n.gate_rows = gate_rows;
  }
  if (branch_weight.defined()) {
    n.branch_weight = branch_weight.data_ptr();
    n.branch_weight_dtype = dtype_code(branch_weight.scalar_type());
  }
  n.scale = (float)scale;
  n.eps = (float)eps;
  return n;
}

// The inputs of a call as the kernels take them; what is not given is undefined.
struct NormInputs {
  at::Tensor x, branch, gate, weight, branch_weight;  // rows, rows, rows, vectors
  int64_t gate_rows;
  double scale, eps;
  fb_norm_t c() const { return norm_of(x, branch, gate, weight, branch_weight, gate_rows, scale, eps); }
};
NormInputs norm_inputs(const at::Tensor& x, const std::optional<at::Tensor>& branch,
                       const std::optional<at::Tensor>& gate, const at::Tensor& weight,
                       const std::optional<at::Tensor>& branch_weight, int64_t gate_rows, double scale,
                       double eps) {
  NormInputs n{as_rows(x), {}, {}, weight.contiguous(), {}, gate_rows, scale, eps};
  if (branch) n.branch = as_rows(*branch);
  if (gate) n.gate = gate->reshape({-1, x.size(-1)}).contiguous();
  if (branch_weight) n.branch_weight = branch_weight->contiguous();
  return n;
}

// stream, normed (of x's shape), stats.
std::vector<at::Tensor> norm_forward(const NormInputs& n, const at::Tensor& x, bool stats) {
  c10::DeviceGuard guard(x.device());
  const auto like = x.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor h = n.branch.defined() ? at::empty(x.sizes(), like) : x;
  at::Tensor y = at::empty(x.sizes(), like);
  at::Tensor st = stats ? at::empty({n.x.size(0), 2}, x.options().dtype(at::kFloat)) : at::Tensor();
  if (x.numel() == 0) return {h, y, st};
  const fb_norm_t c = n.c();
  check(fb_residual_norm(&c, n.branch.defined() ? h.data_ptr() : nullptr, y.data_ptr(),
                         stats ? static_cast<float*>(st.data_ptr()) : nullptr, stream_of(x)));
  return {h, y, st};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& x,
                                                const std::optional<at::Tensor>& branch,
                                                const std::optional<at::Tensor>& gate,
                                                const at::Tensor& weight,
                                                const std::optional<at::Tensor>& branch_weight,
                                                int64_t gate_rows, double scale, double eps) {
    const NormInputs n = norm_inputs(x, branch, gate, weight, branch_weight, gate_rows, scale, eps);
    const auto r = norm_forward(n, x, true);
    ctx->save_for_backward({n.x, n.branch, n.gate, n.weight, n.branch_weight, r[2]});
    ctx->saved_data["gate_rows"] = gate_rows;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["sizes"] = x.sizes().vec();
    if (gate) ctx->saved_data["gate"] = gate->sizes().vec();
    ctx->set_materialize_grads(false);
    // without a branch the stream is x, as a result, so that its gradient is added here, in fp32
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_derivative("residual_norm has no second derivative");
    const auto s = ctx->get_saved_variables();
    const NormInputs n{s[0], s[1], s[2], s[3], s[4], ctx->saved_data["gate_rows"].toInt(),
                       ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble()};
    const at::Tensor& x = n.x;
    c10::DeviceGuard guard(x.device());
    at::Tensor gh = grads[0], gy = grads[1];
    if (gy.defined()) gy = gy.contiguous();
    if (gh.defined()) gh = gh.contiguous();
    at::Tensor out[5];
    const at::Tensor* of[5] = {&n.x, &n.branch, &n.gate, &n.weight, &n.branch_weight};
    for (int i = 0, edge = 0; i < 5; ++i) {  // autograd counts the inputs that there are
      if (!of[i]->defined() || !ctx->needs_input_grad(edge++)) continue;
      const auto sizes = i < 2    ? ctx->saved_data["sizes"].toIntVector()
                         : i == 2 ? ctx->saved_data["gate"].toIntVector()
                                  : of[i]->sizes().vec();
      out[i] = at::empty(sizes, of[i]->options().memory_format(at::MemoryFormat::Contiguous));
      if (x.size(0) == 0) out[i].zero_();
    }
    if (x.size(0)) {
      const auto ptr = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      const fb_norm_t c = n.c();
      const size_t need = fb_residual_norm_grad_workspace_bytes(&c);
      const at::Tensor ws = scratch(need, x);
      check(fb_residual_norm_grad(&c, static_cast<const float*>(s[5].data_ptr()), ptr(gh), ptr(gy),
                                  ptr(out[0]), ptr(out[1]), ptr(out[3]), ptr(out[4]), ptr(out[2]),
                                  ws.data_ptr(), need, stream_of(x)));
    }
    return {out[0], out[1], out[2], out[3], out[4], at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// stream, normed.
std::tuple<at::Tensor, at::Tensor> residual_norm(const at::Tensor& x, const at::Tensor& weight,
                                                 const std::optional<at::Tensor>& branch,
                                                 const std::optional<at::Tensor>& gate, double scale,
                                                 const std::optional<at::Tensor>& branch_weight,
                                                 double eps) {
  not_recorded();
  want(x.defined() && plain(x), "x must be a tensor on a ROCm GPU");
  want(dtype_code(x.scalar_type()) >= 0, "x must be float16, bfloat16 or float32");
  want(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 32768,
       "x must be [..., width], a width of at most 32768");
  const int64_t d = x.size(-1);
  const auto vector = [&](const at::Tensor& t, const char* what) {
    want_plain(t, x, what);
    want(t.dim() == 1 && t.size(0) == d &&
             (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat),
         what);
  };
  vector(weight, "weight must be [width], of x's dtype or float32");
  if (branch_weight) vector(*branch_weight, "branch_weight must be [width], of x's dtype or float32");
  want(branch || (!gate && !branch_weight), "gate and branch_weight need a branch");
  want(std::isfinite(scale) && std::isfinite(eps) && eps >= 0,
       "scale must be finite, eps finite and not negative");
  const int64_t M = x.numel() / d;
  want(M <= INT32_MAX, "too many rows");
  if (branch) {
    want_plain(*branch, x, "branch must be a tensor on x's GPU");
    want(branch->sizes() == x.sizes() && branch->scalar_type() == x.scalar_type(),
         "branch must have x's shape and dtype");
  }
  int64_t gate_rows = 1;
  if (gate) {
    want_plain(*gate, x, "gate must be a tensor on x's GPU");
    want(gate->scalar_type() == x.scalar_type() || gate->scalar_type() == at::kFloat,
         "gate must be of x's dtype or float32");
    const char* what = "gate must be [width], or have x's shape but for leading dimensions of 1 from some "
                       "one on to the last but one (expand others)";
    want(gate->dim() >= 1 && gate->dim() <= x.dim() && gate->size(-1) == d, what);
    // of the leading dimensions the gate has the first k, and one of all others: rows that follow each
    // other share one of its rows
    const int64_t missing = x.dim() - gate->dim();
    const auto size = [&](int64_t i) { return i < missing ? 1 : gate->size(i - missing); };
    int64_t k = 0, rows = 1;
    while (k + 1 < x.dim() && size(k) == x.size(k)) rows *= x.size(k++);
    for (int64_t i = k; i + 1 < x.dim(); ++i) want(size(i) == 1, what);
    gate_rows = std::max<int64_t>(1, rows ? M / rows : 1);
  }
  const auto grad = [](const std::optional<at::Tensor>& t) { return t && t->requires_grad(); };
  if (at::GradMode::is_enabled()) capturable({x, branch, gate, weight, branch_weight});
  std::vector<at::Tensor> r;
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || grad(branch) ||
                                     grad(gate) || grad(branch_weight)))
    r = ResidualNorm::apply(x, branch, gate, weight, branch_weight, gate_rows, scale, eps);
  else
    r = norm_forward(norm_inputs(x, branch, gate, weight, branch_weight, gate_rows, scale, eps), x, false);
  return {r[0], r[1]};
}

// A 16-bit matrix as the head's products take it: 16-byte aligned, rows a multiple of 8 values apart,
// with zeros up to the next multiple of 8 values of a row.
at::Tensor head_side(const at::Tensor& t) {
  const int64_t K = t.size(1);
  if (K % 8 == 0 && row_stride(t) % 8 == 0 && row_stride(t) >= K && row_stride(t) <= (1 << 20) &&
      !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u))
    return t;
  const int64_t ld = (K + 7) / 8 * 8;
  at::Tensor out =
      at::empty({t.size(0), ld}, t.options().memory_format(at::MemoryFormat::Contiguous));
  check(fb_pad_rows(t.data_ptr(), row_stride(t), t.size(0), (int32_t)K, out.data_ptr(), ld,
                    stream_of(t)));
  return out;
}

// logprob, entropy (of the tokens' shape), stats for rows x; and x and w as the products take them (the
// gradient's take them again: a copy, where one was made, is kept for it).
std::vector<at::Tensor> head_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& token,
                                     at::IntArrayRef sizes) {
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), V = w.size(0);
  const auto f = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor lp = at::empty(sizes, f), ent = at::empty(sizes, f), st = at::empty({M, 2}, f);
  if (M == 0) return {lp, ent, st, x, w};
  const at::Tensor xs = head_side(x), ws_ = head_side(w);
  const size_t need = fb_head_logprobs_workspace_bytes(M, (int32_t)K, (int32_t)V);
  const at::Tensor ws = scratch(need, x);
  check(fb_head_logprobs(xs.data_ptr(), row_stride(xs), ws_.data_ptr(), row_stride(ws_),
                         dtype_code(x.scalar_type()), M, (int32_t)K, (int32_t)V,
                         static_cast<const int64_t*>(token.data_ptr()),
                         static_cast<float*>(lp.data_ptr()), static_cast<float*>(ent.data_ptr()),
                         static_cast<float*>(st.data_ptr()), ws.data_ptr(), need, stream_of(x)));
  return {lp, ent, st, xs, ws_};
}

const float* f32_of(const at::Tensor& t) {
  return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr;
}

struct HeadLogprobs : torch::autograd::Function<HeadLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& hidden, const at::Tensor& weight,
                                                const at::Tensor& token,
                                                const std::vector<int64_t>& sizes) {
    const at::Tensor x = as_rows(hidden), w = as_rows(weight);
    const auto r = head_forward(x, w, token, sizes);
    ctx->save_for_backward({x, w, token, r[1], r[2], r[3], r[4]});
    ctx->saved_data["sizes"] = hidden.sizes().vec();
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_derivative("head_logprobs has no second derivative");
    const auto s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &w = s[1], &token = s[2], &ent = s[3], &st = s[4];
    const at::Tensor &xs = s[5], &ws_ = s[6];
    c10::DeviceGuard guard(x.device());
    at::Tensor g[2];
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
    const int64_t M = x.size(0), K = x.size(1), V = w.size(0);
    at::Tensor gx, gw;
    if (ctx->needs_input_grad(0))
      gx = at::empty(ctx->saved_data["sizes"].toIntVector(),
                     x.options().memory_format(at::MemoryFormat::Contiguous));
    if (ctx->needs_input_grad(1)) {
      gw = at::empty(w.sizes(), w.options().memory_format(at::MemoryFormat::Contiguous));
      if (M == 0) gw.zero_();
    }
    if (M) {
      const size_t need = fb_head_logprobs_grad_workspace_bytes(M, (int32_t)K, (int32_t)V,
                                                                gx.defined(), gw.defined());
      const at::Tensor ws = scratch(need, x);
      check(fb_head_logprobs_grad(
          xs.data_ptr(), row_stride(xs), ws_.data_ptr(), row_stride(ws_), dtype_code(x.scalar_type()),
          M, (int32_t)K, (int32_t)V, static_cast<const int64_t*>(token.data_ptr()), f32_of(st),
          f32_of(ent), f32_of(g[0]), f32_of(g[1]), gx.defined() ? gx.data_ptr() : nullptr,
          gw.defined() ? gw.data_ptr() : nullptr, ws.data_ptr(), need, stream_of(x)));
    }
    return {gx, gw, at::Tensor(), at::Tensor()};
  }
};

// A packed head: its logits are fb_gemv's or fb_gemm's, in fp32, for as many rows at once as they take
// half a GiB.
constexpr int64_t kMostLogits = 1 << 27;

struct Packed {
  at::Tensor wdev;
  int64_t N, K, fmt, fwht;
  bool f16_exact, bf16_exact;
};

fb_shape_t packed_shape(const Packed& p, int64_t rows, int xdt, int ydt) {
  fb_shape_t s{};
  s.N = (int32_t)p.N;
  s.K = (int32_t)((p.K + 127) / 128 * 128);
  s.B = (int32_t)rows;
  s.group = p.fmt == FB_FMT_E2M1 ? 32 : 128;
  s.fmt = (int32_t)p.fmt;
  s.fwht_block = (int32_t)p.fwht;
  s.x_dtype = xdt;
  s.y_dtype = ydt;
  return s;
}

// x [M, K] as the kernels take it: fp16 for GF4 and rotations, else fp16 or bf16, rows of the packed K.
at::Tensor packed_rows(const Packed& p, const at::Tensor& x) {
  const int xdt = dtype_code(x.scalar_type());
  int kdt = xdt == FB_DT_F32 ? FB_DT_BF16 : xdt;
  if (p.fmt != FB_FMT_E2M1 || p.fwht) kdt = FB_DT_F16;
  want(p.fmt != FB_FMT_E2M1 || kdt != FB_DT_F16 || p.f16_exact,
       "the head's E2M1 scales do not decode exactly to float16: pass bfloat16 hidden states");
  const int64_t kp = (p.K + 127) / 128 * 128;
  const at::Tensor c = x.contiguous();
  if (kdt == xdt && kp == p.K && !(reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u)) return c;
  at::Tensor out =
      at::empty({x.size(0), kp}, x.options().dtype(kdt == FB_DT_F16 ? at::kHalf : at::kBFloat16));
  check(fb_cast_rows(c.data_ptr(), xdt, (int32_t)x.size(0), (int32_t)p.K, out.data_ptr(), kdt, (int32_t)kp,
                     stream_of(x)));
  return out;
}

// fp32 logits of rows r .. r + n - 1 of xk into y [>= n, N].
void packed_logits(const Packed& p, const at::Tensor& xk, int64_t r, int64_t n, const at::Tensor& y) {
  fb_shape_t s = packed_shape(p, n, dtype_code(xk.scalar_type()), FB_DT_F32);
  const void* x = static_cast<const char*>(xk.data_ptr()) + r * xk.size(1) * 2;
  if (n <= kMaxGemvBatch) {
    const size_t need = fb_workspace_bytes(&s);
    const at::Tensor ws = need ? scratch(need, xk) : at::Tensor();
    check(fb_gemv(p.wdev.data_ptr(), x, y.data_ptr(), &s, ptr_or_null(ws, need), need, stream_of(xk)));
  } else {
    const size_t need = fb_gemm_workspace_bytes(&s);
    const at::Tensor ws = need ? scratch(need, xk) : at::Tensor();
    check(fb_gemm(p.wdev.data_ptr(), x, y.data_ptr(), &s, nullptr, 0, ptr_or_null(ws, need), need,
                  stream_of(xk)));
  }
}

int64_t packed_piece(const Packed& p, int64_t M) {
  return std::min(M, std::max<int64_t>(16, std::min<int64_t>(kMostLogits / p.N, kGradRows) / 16 * 16));
}

std::vector<at::Tensor> packed_forward(const Packed& p, const at::Tensor& x, const at::Tensor& token,
                                       at::IntArrayRef sizes) {
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0);
  const auto f = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor lp = at::empty(sizes, f), ent = at::empty(sizes, f), st = at::empty({M, 3}, f);
  if (M == 0) return {lp, ent, st};
  const at::Tensor xk = packed_rows(p, x);
  const int64_t step = packed_piece(p, M);
  const at::Tensor y = at::empty({step, p.N}, f);
  for (int64_t r = 0; r < M; r += step) {
    const int64_t n = std::min(step, M - r);
    packed_logits(p, xk, r, n, y);
    check(fb_token_logprobs(y.data_ptr(), FB_DT_F32, p.N, n, (int32_t)p.N,
                            static_cast<const int64_t*>(token.data_ptr()) + r, 0,
                            static_cast<float*>(lp.data_ptr()) + r,
                            static_cast<float*>(ent.data_ptr()) + r, nullptr, nullptr,
                            static_cast<float*>(st.data_ptr()) + 3 * r, stream_of(x)));
  }
  return {lp, ent, st};
}

// gl W for n rows of fp32 gl [>= n, N] into gx [n, kp], in fp32 terms, as many tokens as fb_grad_x takes
// at once.
void packed_grad_rows(const Packed& p, const at::Tensor& gl, int64_t n, const at::Tensor& gx) {
  at::Tensor sum;
  for (int64_t v = 0; v < p.N; v += kGradVocab) {
    Packed part = p;
    part.N = std::min(kGradVocab, p.N - v);
    const fb_shape_t s = packed_shape(part, n, FB_DT_F16, FB_DT_F32);
    part.N = v;  // of what lies before it, whole tiles of 16 rows
    const fb_shape_t before = packed_shape(part, 1, FB_DT_F16, FB_DT_F32);
    const bool all = s.N == p.N;
    const at::Tensor g = all ? gl : gl.narrow(0, 0, n).narrow(1, v, s.N).contiguous();
    const at::Tensor out = all ? gx : at::empty(gx.sizes(), gx.options().dtype(at::kFloat));
    const size_t need = fb_grad_x_workspace_bytes(&s, p.f16_exact);  // fewer rows may need more
    const at::Tensor ws = scratch(need, gx);
    check(fb_grad_x(static_cast<const char*>(p.wdev.data_ptr()) + (v ? fb_device_bytes(&before) : 0),
                    g.data_ptr(), out.data_ptr(), &s, dtype_code(out.scalar_type()), p.f16_exact,
                    ws.data_ptr(), need, stream_of(gx)));
    if (!all) sum = sum.defined() ? sum.add_(out) : out;
  }
  if (sum.defined()) gx.copy_(sum);
}

struct PackedHeadLogprobs : torch::autograd::Function<PackedHeadLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                const at::Tensor& hidden, const at::Tensor& wdev,
                                                const at::Tensor& token,
                                                const std::vector<int64_t>& sizes, int64_t N, int64_t K,
                                                int64_t fmt, int64_t fwht, bool f16_exact,
                                                bool bf16_exact) {
    const Packed p{wdev, N, K, fmt, fwht, f16_exact, bf16_exact};
    const at::Tensor x = as_rows(hidden);
    const auto r = packed_forward(p, x, token, sizes);
    ctx->saved_data["sizes"] = hidden.sizes().vec();
    ctx->save_for_backward({x, wdev, token, r[1], r[2]});
    ctx->saved_data["head"] = std::vector<int64_t>{N, K, fmt, fwht, f16_exact, bf16_exact};
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_derivative("head_logprobs has no second derivative");
    const auto s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &token = s[2], &ent = s[3], &st = s[4];
    const auto h = ctx->saved_data["head"].toIntVector();
    const Packed p{s[1], h[0], h[1], h[2], h[3], (bool)h[4], (bool)h[5]};
    c10::DeviceGuard guard(x.device());
    at::Tensor g[2];
    for (int i = 0; i < 2; ++i)
      if (grads[i].defined()) g[i] = grads[i].to(at::kFloat).contiguous();
    const int64_t M = x.size(0), kp = (p.K + 127) / 128 * 128;
    at::Tensor gx = at::empty({M, kp}, x.options().memory_format(at::MemoryFormat::Contiguous));
    const int xdt = dtype_code(x.scalar_type());
    const at::Tensor xk = M ? packed_rows(p, x) : at::Tensor();
    // of 16-bit hidden states with the weight in 16 bits too, where it is exact there, not rotated and within
    // that call's limits; else, fp32 hidden states among them, in fp32 terms.  (The 16-bit way would take 775
    // us of fp32 hidden states of 1024 x 32000 x 4096, E2M1, instead of 1,590, and lose 3e-4 to 1.5e-3 of
    // their gradient.)
    const bool exact = p.fmt != FB_FMT_E2M1 || !M ||
                       (xk.scalar_type() == at::kHalf ? p.f16_exact : p.bf16_exact);
    if (M && !p.fwht && exact && xdt != FB_DT_F32 && p.N <= (1 << 24) && M * kp <= (1ll << 33)) {
      fb_shape_t sh = packed_shape(p, M, dtype_code(xk.scalar_type()), FB_DT_F32);
      const size_t need = fb_packed_head_grad_workspace_bytes(&sh);
      const at::Tensor ws = scratch(need, x);
      check(fb_packed_head_grad(p.wdev.data_ptr(), xk.data_ptr(), &sh,
                                static_cast<const int64_t*>(token.data_ptr()), f32_of(st), f32_of(ent),
                                f32_of(g[0]), f32_of(g[1]), gx.data_ptr(), xdt, ws.data_ptr(), need,
                                stream_of(x)));
    } else if (M) {
      const int64_t step = packed_piece(p, M);
      const auto f = x.options().dtype(at::kFloat);
      const at::Tensor y = at::empty({step, p.N}, f), gl = at::empty({step, p.N}, f);
      for (int64_t r = 0; r < M; r += step) {
        const int64_t n = std::min(step, M - r);
        packed_logits(p, xk, r, n, y);
        check(fb_token_logprobs_grad(
            y.data_ptr(), FB_DT_F32, p.N, n, (int32_t)p.N,
            static_cast<const int64_t*>(token.data_ptr()) + r, 0, nullptr, f32_of(st) + 3 * r,
            f32_of(ent) + r, g[0].defined() ? f32_of(g[0]) + r : nullptr,
            g[1].defined() ? f32_of(g[1]) + r : nullptr, nullptr, gl.data_ptr(), stream_of(x)));
        packed_grad_rows(p, gl, n, gx.narrow(0, r, n));
      }
      // rows that nothing comes in for, whose logits may be NaN
      at::Tensor some = at::zeros({M}, token.options().dtype(at::kBool));
      if (g[0].defined())
        some.logical_or_(token.ge(0).logical_and_(token.lt(p.N)).logical_and_(g[0].view({M})));
      if (g[1].defined()) some.logical_or_(g[1].view({M}));
      gx.masked_fill_(some.logical_not_().unsqueeze(1), 0);
    }
    if (kp != p.K) gx = gx.narrow(1, 0, p.K).contiguous();
    return {gx.view(ctx->saved_data["sizes"].toIntVector()), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// x [..., K] and tokens [...]: the flat tokens, after the checks that both kinds of heads share.
at::Tensor head_tokens(const at::Tensor& x, const at::Tensor& tokens, int64_t K,
                                              const at::Tensor& like) {
  not_recorded();
  want(x.defined() && plain(x), "hidden must be a tensor on a ROCm GPU");
  want(x.device() == like.device(), "all tensors must be on one GPU");
  want_tokens(tokens, x);
  want(x.dim() >= 1 && x.size(-1) == K, "hidden must be [..., width] with the head's width");
  want(tokens.sizes() == x.sizes().slice(0, x.dim() - 1),
       "tokens must have hidden's shape without the last dimension");
  want(tokens.numel() <= (1 << 23), "too many tokens");
  return flat_tokens(tokens);
}

// logprob, entropy.
std::tuple<at::Tensor, at::Tensor> head_logprobs(const at::Tensor& hidden, const at::Tensor& weight,
                                                 const at::Tensor& tokens) {
  want(weight.defined() && plain(weight), "the head must be a tensor on a ROCm GPU or packed");
  want(weight.dim() == 2 && weight.size(0) >= 1 && weight.size(0) <= (1 << 24) && weight.size(1) >= 1 &&
           weight.size(1) <= (1 << 20),
       "the head's weight must be [vocab, width], a width of at most 2^20, a vocabulary of at most 2^24");
  const at::Tensor t = head_tokens(hidden, tokens, weight.size(1), weight);
  want((hidden.scalar_type() == at::kHalf || hidden.scalar_type() == at::kBFloat16) &&
           hidden.scalar_type() == weight.scalar_type(),
       "hidden and the head's weight must both be float16 or both bfloat16");
  if (at::GradMode::is_enabled()) capturable({hidden, weight});
  const auto r = at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad())
                     ? HeadLogprobs::apply(hidden, weight, t, tokens.sizes().vec())
                     : head_forward(as_rows(hidden), as_rows(weight), t, tokens.sizes());
  return {r[0], r[1]};
}

std::tuple<at::Tensor, at::Tensor> packed_head_logprobs(const at::Tensor& hidden, const at::Tensor& wdev,
                                                        const at::Tensor& tokens, int64_t N, int64_t K,
                                                        int64_t fmt, int64_t fwht, bool f16_exact,
                                                        bool bf16_exact) {
  want(wdev.defined() && plain(wdev), "the packed head must be on a ROCm GPU");
  const at::Tensor t = head_tokens(hidden, tokens, K, wdev);
  want(dtype_code(hidden.scalar_type()) >= 0, "hidden must be float16, bfloat16 or float32");
  const Packed p{wdev, N, K, fmt, fwht, f16_exact, bf16_exact};
  const fb_shape_t s = packed_shape(p, 1, FB_DT_F16, FB_DT_F32);
  want(fb_device_bytes(&s) && (size_t)wdev.numel() >= fb_device_bytes(&s) && s.K <= kMaxGemmK,
       "the packed head is not of its format's size");
  if (at::GradMode::is_enabled()) capturable({hidden});
  const auto r = at::GradMode::is_enabled() && hidden.requires_grad()
                     ? PackedHeadLogprobs::apply(hidden, wdev, t, tokens.sizes().vec(), N, K, fmt, fwht,
                                                 f16_exact, bf16_exact)
                     : packed_forward(p, as_rows(hidden), t, tokens.sizes());
  return {r[0], r[1]};
}

}  // namespace

PYBIND11_MODULE(_fourbit_torch, m) {
  m.def("linear_forward", &linear_forward);
  m.def("linear_grad_x", &linear_grad_x);
  m.def("linear_grad_bias", &linear_grad_bias);
  m.def("added_bias", &added_bias);
  m.def("cache_append", &cache_append);
  m.def("cache_attention", &cache_attention);
  m.def("cache_evict", &cache_evict);
  m.def("token_logprobs", &token_logprobs);
  m.def("token_embedding", &token_embedding);
  m.def("residual_norm", &residual_norm);
  m.def("head_logprobs", &head_logprobs);
  m.def("packed_head_logprobs", &packed_head_logprobs);
}
