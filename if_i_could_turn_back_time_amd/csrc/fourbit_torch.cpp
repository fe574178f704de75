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
}
