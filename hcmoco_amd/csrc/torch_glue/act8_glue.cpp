// torch.ops.hcmoco.* of the 8-bit training operators: argument checks, buffers and autograd nodes over the C ABI.
//
// In C++ for the reason that bn_act is: a Python autograd.Function and its ctypes calls cost 150 us of host time for a layer norm's
// two directions, more than every kernel of a small batch.  hip_ops.layer_norm / act8_pack / act8_unpack / fp8_* document the
// operators; the errors raised here are the ones they document (TypeError, ValueError, RuntimeError).
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>

#include "hcmoco_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

void* stream_of(const Tensor& t) { return static_cast<void*>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: hip error ", rc, " (", hcm_error_string(rc), ")"); }

int dt_of(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return HCM_DT_F32;
    case at::kBFloat16: return HCM_DT_BF16;
    case at::kHalf: return HCM_DT_F16;
    default: TORCH_CHECK_TYPE(false, name, ": expected float32, bfloat16 or float16, got ", t);
  }
}
int dt_of(const Tensor& t, const char* name) { return t.defined() ? dt_of(t.scalar_type(), name) : 0; }

// what an operator reads: a 16- or 32-bit floating ROCm tensor, on the device of the first
void check_float(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda(), "hcmoco_amd.", name, " needs ROCm device tensors (no CPU fallback exists)");
  dt_of(t, name);
  TORCH_CHECK_VALUE(t.device() == first.device(), name, ": tensors on ", first.device(), " and on ", t.device());
}
void check_bytes(const Tensor& t, int64_t rows, int64_t width, const Tensor& first, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.scalar_type() == at::kByte && t.dim() == 2 && t.size(0) == rows && t.size(1) == width && t.is_contiguous() &&
                        t.device() == first.device(),
                    name, ": the 8-bit buffers do not hold a tensor of this shape on ", first.device());
}

Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
uint8_t* bytes(const Tensor& t) { return t.defined() ? t.data_ptr<uint8_t>() : nullptr; }

// x [..., C] as rows; a 2-D column slice is read where it lies
struct Rows { Tensor t; int64_t rows, ld; int cols; };
Rows rows_of(const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, name, ": the last axis must have at least one element");
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  TORCH_CHECK_VALUE(cols <= INT32_MAX - 16384 && rows < (1ll << 31) - 8192 && rows * ((cols + 127) / 128) < (1ll << 30), name, ": ", rows, " rows of ", cols,
                    " values are too many (at most 2^30 blocks of 128)");
  if (x.is_contiguous()) return {x, rows, cols, (int)cols};
  if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= cols) return {x, rows, x.stride(0), (int)cols};
  return {x.contiguous(), rows, cols, (int)cols};
}

struct Packed { Tensor q, scale; };
Packed packed_buffers(int64_t rows, int64_t cols, const Tensor& like) {
  const auto o = like.options().dtype(at::kByte);
  return {at::empty({rows, hcm_act8_pitch(cols)}, o), at::empty({rows, hcm_act8_scale_pitch(cols)}, o)};
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s(sizes.begin(), sizes.end());
  s.back() = last;
  return s;
}

Tensor workspace(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

// What the backward pass gets back of a tensor it saved.  A saved-tensor hook may return it in another layout, on other memory
// (save_on_cpu: a contiguous copy of what was a column slice), so nothing but the size is taken from the forward pass, and that is checked.
Tensor restored(const Tensor& t, at::ScalarType dtype, at::IntArrayRef sizes, const Tensor& dy, const char* name) {
  TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.scalar_type() == dtype && t.sizes() == sizes && t.device() == dy.device(), name,
              ": a saved tensor of type ", dtype, " and size ", sizes, " on ", dy.device(), " came back from its hook as something else");
  return t;
}
// the same for a buffer, as it was allocated: contiguous, the 8-bit ones on a 16-byte border
Tensor restored_buffer(const Tensor& t, at::ScalarType dtype, at::IntArrayRef sizes, const Tensor& dy, const char* name) {
  const Tensor c = restored(t, dtype, sizes, dy, name).contiguous();
  return dtype == at::kByte && ((uintptr_t)c.data_ptr() & 15) ? c.clone() : c;
}

// A backward pass that is itself recorded (create_graph) has no second derivative: asking for one raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>("hcmoco 8-bit operators have no second derivative", (int64_t)grads.size());
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  at::AutoGradMode on(true);
  return (*node)(std::move(grads));
}

// ------------------------------------------------------------------------------------------------------------
// act8
// ------------------------------------------------------------------------------------------------------------
Packed pack_raw(const Rows& r, const char* name) {
  Packed p = packed_buffers(r.rows, r.cols, r.t);
  if (r.rows)
    check_rc(hcm_act8_pack(r.t.data_ptr(), dt_of(r.t, name), r.rows, r.cols, r.ld, bytes(p.q), p.q.size(1), bytes(p.scale), p.scale.size(1), stream_of(r.t)),
             "hcm_act8_pack");
  return p;
}

std::tuple<Tensor, Tensor> act8_pack(const Tensor& x) {
  check_float(x, x, "act8_pack");
  at::AutoGradMode off(false);
  const c10::DeviceGuard guard(x.device());
  Packed p = pack_raw(rows_of(x, "act8_pack"), "act8_pack");
  return {p.q, p.scale};
}

Tensor act8_unpack(const Tensor& q, const Tensor& scale, at::IntArrayRef shape, at::ScalarType dtype) {
  const int dt = dt_of(dtype, "act8_unpack");
  TORCH_CHECK_VALUE(!shape.empty() && shape.back() > 0 && shape.back() <= INT32_MAX - 16384, "act8_unpack: the last axis must have at least one element");
  const int64_t cols = shape.back(), rows = c10::multiply_integers(shape) / cols;
  check_bytes(q, rows, hcm_act8_pitch(cols), q, "act8_unpack");
  check_bytes(scale, rows, hcm_act8_scale_pitch(cols), q, "act8_unpack");
  const c10::DeviceGuard guard(q.device());
  Tensor x = at::empty(shape, q.options().dtype(dtype));
  if (rows)
    check_rc(hcm_act8_unpack(bytes(q), q.size(1), bytes(scale), scale.size(1), rows, (int)cols, x.data_ptr(), dt, stream_of(q)), "hcm_act8_unpack");
  return x;
}

// ------------------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------------------
struct NormOut { Tensor y, stats, a, scale; Rows r; };

NormOut norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, bool need, bool act8) {
  NormOut o;
  o.r = rows_of(x, "layer_norm");
  const Rows& r = o.r;
  o.y = at::empty(x.sizes(), x.options());
  Packed p;
  float* stats = nullptr;
  if (need) {
    o.stats = at::empty({2, r.rows}, x.options().dtype(at::kFloat));
    stats = o.stats.data_ptr<float>();
    if (act8) p = packed_buffers(r.rows, r.cols, x);
  }
  o.a = need && act8 ? p.q : r.t;
  o.scale = p.scale;
  if (r.rows)
    check_rc(hcm_layer_norm_forward(r.t.data_ptr(), dt_of(x, "layer_norm"), r.rows, r.cols, r.ld, ptr(w), dt_of(w, "layer_norm"), ptr(b),
                                    dt_of(b, "layer_norm"), (float)eps, o.y.data_ptr(), stats, need ? stats + r.rows : nullptr, bytes(p.q),
                                    p.q.defined() ? p.q.size(1) : 0, bytes(p.scale), p.q.defined() ? p.scale.size(1) : 0, stream_of(x)),
             "hcm_layer_norm_forward");
  return o;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool act8) {
    const Tensor w = value(weight), b = value(bias);
    NormOut o = norm_forward(x, w, b, eps, true, act8);
    const bool nx = x.requires_grad(), nw = w.defined() && w.requires_grad(), nb = b.defined() && b.requires_grad();
    ctx->save_for_backward({o.a, o.scale, o.stats, w});
    ctx->saved_data["m"] = std::vector<int64_t>{o.r.rows, o.r.cols, act8, nx, nw, nb, w.defined() ? (int64_t)w.scalar_type() : -1,
                                                b.defined() ? (int64_t)b.scalar_type() : 0};
    return o.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    const int64_t rows = m[0];
    const int cols = (int)m[1];
    const bool act8 = m[2], nx = m[3], nw = m[4], nb = m[5];
    Tensor dx, dw, db;
    {
      at::AutoGradMode off(false);
      const Tensor dy = grads[0].contiguous();
      const c10::DeviceGuard guard(dy.device());
      Rows x{};
      Packed p;
      if (act8) {
        p.q = restored_buffer(saved[0], at::kByte, {rows, hcm_act8_pitch(cols)}, dy, "layer_norm");
        p.scale = restored_buffer(saved[1], at::kByte, {rows, hcm_act8_scale_pitch(cols)}, dy, "layer_norm");
      } else {
        x = rows_of(restored(saved[0], dy.scalar_type(), dy.sizes(), dy, "layer_norm"), "layer_norm");
      }
      const Tensor stats = restored_buffer(saved[2], at::kFloat, {2, rows}, dy, "layer_norm");
      const Tensor w = m[6] < 0 ? Tensor() : restored_buffer(saved[3], (at::ScalarType)m[6], {cols}, dy, "layer_norm");
      dx = at::empty_like(dy);
      if (nw) dw = at::empty({cols}, w.options());
      if (nb) db = at::empty({cols}, dy.options().dtype((at::ScalarType)m[7]));
      if (rows) {
        const size_t n = hcm_layer_norm_backward_workspace_bytes(rows, cols);
        const Tensor ws = workspace(n, dy);
        const float* st = stats.data_ptr<float>();
        check_rc(hcm_layer_norm_backward(ptr(x.t), x.ld, bytes(p.q), act8 ? p.q.size(1) : 0, bytes(p.scale), act8 ? p.scale.size(1) : 0, dy.data_ptr(),
                                         dt_of(dy, "layer_norm"), rows, cols, ptr(w), dt_of(w, "layer_norm"), st, st + rows, dx.data_ptr(), ptr(dw), ptr(db),
                                         dt_of(db, "layer_norm"), ptr(ws), n, stream_of(dy)),
                 "hcm_layer_norm_backward");
      } else {
        if (nw) dw.zero_();
        if (nb) db.zero_();
      }
      if (!nx) dx = Tensor();
    }
    return once({dx, dw, db, Tensor(), Tensor()});
  }
};

void check_vector(const Tensor& p, const Tensor& x, int64_t n, const char* name, const char* what) {
  if (!p.defined()) return;
  check_float(p, x, name);
  TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == n && p.is_contiguous(), name, ": ", what, " must be a contiguous vector of ", n, " values");
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Forward-mode differentiation: these operators have no rule for it, and a dual tensor that no backward graph records would lose its
// tangent without a word (a missing tangent reads as zero).
void check_no_tangent(std::initializer_list<const Tensor*> inputs, const char* name) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative");
}

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, bool act8) {
  const Tensor w = value(weight), b = value(bias);
  check_float(x, x, "layer_norm");
  TORCH_CHECK_VALUE(x.dim() > 0, "layer_norm: x needs at least one axis");
  check_vector(w, x, x.size(-1), "layer_norm", "weight");
  check_vector(b, x, x.size(-1), "layer_norm", "bias");
  TORCH_CHECK_VALUE(x.size(-1) < (1 << 27), "layer_norm: rows of at most 2^27 - 1 values, got ", x.size(-1));
  TORCH_CHECK_VALUE(x.size(-1) <= 16384 || x.numel() / x.size(-1) < (1 << 22), "layer_norm: fewer than 2^22 rows of over 16384 values, got ",
                    x.numel() / x.size(-1));
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative");
  check_no_tangent({&x, &w, &b}, "layer_norm");
  const c10::DeviceGuard guard(x.device());
  if (!at::GradMode::is_enabled() || !(wants_grad(x) || wants_grad(w) || wants_grad(b))) return norm_forward(x, w, b, eps, false, false).y;
  return LayerNorm::apply(x, weight, bias, eps, act8);
}

// ------------------------------------------------------------------------------------------------------------
// linear layers on 8-bit blocks
// ------------------------------------------------------------------------------------------------------------
constexpr int64_t kMaxSide = 1 << 22;

std::tuple<Tensor, Tensor, Tensor, Tensor> fp8_weight(const Tensor& weight) {
  check_float(weight, weight, "fp8_weight");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) > 0 && weight.size(0) <= kMaxSide && weight.size(1) > 0 && weight.size(1) <= kMaxSide,
                    "fp8_weight: expected [N, K] with both in 1..2^22, got ", weight.sizes());
  at::AutoGradMode off(false);
  const c10::DeviceGuard guard(weight.device());
  const Rows r = rows_of(weight, "fp8_weight");
  const int64_t N = r.rows, K = r.cols;
  const auto o = weight.options().dtype(at::kByte).requires_grad(false);
  const Tensor q = at::empty({N, hcm_act8_pitch(K)}, o), qt = at::empty({K, hcm_act8_pitch(N)}, o);
  const Tensor scale = at::empty({(N + 127) / 128, hcm_act8_scale_pitch(K)}, o), scale_t = at::empty({(K + 127) / 128, hcm_act8_scale_pitch(N)}, o);
  check_rc(hcm_fp8_weight_pack(r.t.data_ptr(), dt_of(weight, "fp8_weight"), (int)N, (int)K, r.ld, bytes(q), q.size(1), bytes(scale), scale.size(1), bytes(qt),
                               qt.size(1), bytes(scale_t), scale_t.size(1), stream_of(weight)),
           "hcm_fp8_weight_pack");
  return {q, scale, qt, scale_t};
}

// y [M, N] = X W^T + bias on buffers of the pitches of K, everything checked by the caller; `like`: the device
Tensor product(const uint8_t* xq, const uint8_t* xs, int64_t M, const uint8_t* wq, const uint8_t* ws, int64_t N, int64_t K, const Tensor& bias,
               at::IntArrayRef shape, at::ScalarType dtype, const Tensor& like) {
  Tensor y = at::empty(shape, like.options().dtype(dtype));
  if (M) {
    const int dt = dt_of(dtype, "fp8_matmul");
    const size_t n = hcm_fp8_matmul_workspace_bytes((int)M, (int)N, (int)K);
    const Tensor work = workspace(n, like);
    const int64_t pitch = hcm_act8_pitch(K), sp = hcm_act8_scale_pitch(K);
    check_rc(hcm_fp8_matmul(xq, pitch, xs, sp, wq, pitch, ws, sp, ptr(bias), dt_of(bias, "fp8_matmul"), (int)M, (int)N, (int)K, y.data_ptr(), dt, ptr(work),
                            n, stream_of(like)),
             "hcm_fp8_matmul");
  }
  return y;
}

// the four buffers of a laid-out weight [N, K]
void check_weight(const Tensor& wq, const Tensor& ws, int64_t N, int64_t K, const Tensor& x, const char* name) {
  TORCH_CHECK_VALUE(N > 0 && N <= kMaxSide && K > 0 && K <= kMaxSide, name, ": expected a weight [N, K] with both in 1..2^22");
  check_bytes(wq, N, hcm_act8_pitch(K), x, name);
  check_bytes(ws, (N + 127) / 128, hcm_act8_scale_pitch(K), x, name);
}

void check_width(int64_t K, int64_t w_cols, const char* name) {
  TORCH_CHECK_VALUE(w_cols == K, name, ": a weight of ", w_cols, " columns does not go with ", K, " values a row");
}

Tensor fp8_matmul(const Tensor& q, const Tensor& scale, at::IntArrayRef shape, const Tensor& wq, const Tensor& ws, at::IntArrayRef w_shape,
                  const OptTensor& bias, at::ScalarType dtype) {
  dt_of(dtype, "fp8_matmul");
  TORCH_CHECK_VALUE(!shape.empty() && shape.back() > 0, "fp8_matmul: the last axis must have at least one element");
  TORCH_CHECK_VALUE(w_shape.size() == 2, "fp8_matmul: a weight has two axes");
  const int64_t K = shape.back(), M = c10::multiply_integers(shape) / K, N = w_shape[0];
  check_width(K, w_shape[1], "fp8_matmul");
  check_bytes(q, M, hcm_act8_pitch(K), q, "fp8_matmul");
  check_bytes(scale, M, hcm_act8_scale_pitch(K), q, "fp8_matmul");
  check_weight(wq, ws, N, K, q, "fp8_matmul");
  TORCH_CHECK_VALUE(M <= INT32_MAX - 512, "fp8_matmul: too many rows");
  const Tensor b = value(bias);
  check_vector(b, q, N, "fp8_matmul", "bias");
  const c10::DeviceGuard guard(q.device());
  return product(bytes(q), bytes(scale), M, bytes(wq), bytes(ws), N, K, b, with_last(shape, N), dtype, q);
}

// Where the parts of a laid-out weight lie: in the four tensors of an Fp8Weight, or one behind the other in one buffer (a training step
// lays its weight out anew on every call, and four allocations would cost more host time than the launch).
struct Weight8 {
  Tensor first, second;              // what the backward pass keeps: the buffer; or qt and scale_t
  const uint8_t *q, *scale, *qt, *scale_t;
};
int64_t weight_bytes(int64_t N, int64_t K) {
  return N * hcm_act8_pitch(K) + K * hcm_act8_pitch(N) + (N + 127) / 128 * hcm_act8_scale_pitch(K) + (K + 127) / 128 * hcm_act8_scale_pitch(N);
}
Weight8 weight_in(const Tensor& buffer, int64_t N, int64_t K) {
  Weight8 w;
  w.first = buffer;
  w.q = bytes(buffer);
  w.qt = w.q + N * hcm_act8_pitch(K);
  w.scale = w.qt + K * hcm_act8_pitch(N);
  w.scale_t = w.scale + (N + 127) / 128 * hcm_act8_scale_pitch(K);
  return w;
}
Weight8 lay_out(const Tensor& weight) {
  const Rows r = rows_of(weight, "fp8_linear");
  const int64_t N = r.rows, K = r.cols;
  TORCH_CHECK_VALUE(N > 0 && N <= kMaxSide && K <= kMaxSide, "fp8_linear: expected a weight [N, K] with both in 1..2^22, got ", weight.sizes());
  Weight8 w = weight_in(workspace(weight_bytes(N, K), weight), N, K);
  check_rc(hcm_fp8_weight_pack(r.t.data_ptr(), dt_of(weight, "fp8_linear"), (int)N, (int)K, r.ld, (uint8_t*)w.q, hcm_act8_pitch(K), (uint8_t*)w.scale,
                               hcm_act8_scale_pitch(K), (uint8_t*)w.qt, hcm_act8_pitch(N), (uint8_t*)w.scale_t, hcm_act8_scale_pitch(N), stream_of(weight)),
           "hcm_fp8_weight_pack");
  return w;
}

// Q(x) W^T + bias for x as it comes.  `packed`: Q(x) is wanted too, its scales behind its values in one buffer.
Tensor linear_forward(const Rows& r, const uint8_t* wq, const uint8_t* ws, int64_t N, const Tensor& bias, at::IntArrayRef shape, Tensor* packed) {
  const bool few = hcm_fp8_rows_supported(r.rows, r.cols);
  const int64_t pitch = hcm_act8_pitch(r.cols), sp = hcm_act8_scale_pitch(r.cols);
  Tensor buffer;
  uint8_t *q = nullptr, *scale = nullptr;
  if (packed || !few) {
    buffer = at::empty({r.rows * (pitch + sp)}, r.t.options().dtype(at::kByte));
    q = bytes(buffer);
    scale = q + r.rows * pitch;
  }
  if (packed) *packed = buffer;
  const int dt = dt_of(r.t, "fp8_linear");
  if (!few) {
    if (r.rows) check_rc(hcm_act8_pack(r.t.data_ptr(), dt, r.rows, r.cols, r.ld, q, pitch, scale, sp, stream_of(r.t)), "hcm_act8_pack");
    return product(q, scale, r.rows, wq, ws, N, r.cols, bias, shape, r.t.scalar_type(), r.t);
  }
  Tensor y = at::empty(shape, r.t.options());
  check_rc(hcm_fp8_rows(r.t.data_ptr(), dt, r.ld, wq, pitch, ws, sp, ptr(bias), dt_of(bias, "fp8_linear"), (int)r.rows, (int)N, r.cols, y.data_ptr(), q, scale,
                        stream_of(r.t)),
           "hcm_fp8_rows");
  return y;
}

struct Fp8Linear : public torch::autograd::Function<Fp8Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, const Weight8& W, int64_t N) {
    const Tensor w = value(weight), b = value(bias);
    const Rows r = rows_of(x, "fp8_linear");
    const bool nx = wants_grad(x), nw = wants_grad(w);
    Tensor packed;
    Tensor y = linear_forward(r, W.q, W.scale, N, b, with_last(x.sizes(), N), nw ? &packed : nullptr);
    // x itself is not kept: the 8-bit operand of this product is the checkpoint that the weight's gradient reads
    ctx->save_for_backward({packed, nx ? W.first : Tensor(), nx ? W.second : Tensor()});
    std::vector<int64_t> m{r.rows, N, r.cols, nx, nw, wants_grad(b), nw ? (int64_t)w.scalar_type() : 0, b.defined() ? (int64_t)b.scalar_type() : 0,
                           !W.second.defined()};
    m.insert(m.end(), x.sizes().begin(), x.sizes().end());
    ctx->saved_data["m"] = std::move(m);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto m = ctx->saved_data["m"].toIntVector();
    const at::IntArrayRef shape(m.data() + 9, m.size() - 9);
    const int64_t M = m[0], N = m[1], K = m[2];
    const bool nx = m[3], nw = m[4], nb = m[5];
    Tensor dx, dw, db;
    {
      at::AutoGradMode off(false);
      Tensor dy = grads[0].contiguous();
      if ((uintptr_t)dy.data_ptr() & 15) dy = dy.clone();        // a view that begins anywhere: hcm_fp8_wgrad reads 16-byte pieces
      const c10::DeviceGuard guard(dy.device());
      if (nx) {
        Weight8 W;
        if (m[8]) {
          W = weight_in(restored_buffer(saved[1], at::kByte, {weight_bytes(N, K)}, dy, "fp8_linear"), N, K);
        } else {
          W.first = restored_buffer(saved[1], at::kByte, {K, hcm_act8_pitch(N)}, dy, "fp8_linear");
          W.second = restored_buffer(saved[2], at::kByte, {(K + 127) / 128, hcm_act8_scale_pitch(N)}, dy, "fp8_linear");
          W.qt = bytes(W.first);
          W.scale_t = bytes(W.second);
        }
        dx = linear_forward({dy, M, N, (int)N}, W.qt, W.scale_t, K, Tensor(), shape, nullptr);
      }
      if (nw) dw = at::empty({N, K}, dy.options().dtype((at::ScalarType)m[6]));
      if (nb) db = at::empty({N}, dy.options().dtype((at::ScalarType)m[7]));
      if ((nw || nb) && M) {
        const int dt = dt_of(dy, "fp8_linear");
        const size_t n = hcm_fp8_wgrad_workspace_bytes(M, (int)N, (int)K, dt, nw);
        const Tensor work = workspace(n, dy);
        const Tensor packed = nw ? restored_buffer(saved[0], at::kByte, {M * (hcm_act8_pitch(K) + hcm_act8_scale_pitch(K))}, dy, "fp8_linear") : Tensor();
        const uint8_t* q = bytes(packed);
        check_rc(hcm_fp8_wgrad(q, hcm_act8_pitch(K), nw ? q + M * hcm_act8_pitch(K) : nullptr, hcm_act8_scale_pitch(K), dy.data_ptr(), dt, M, (int)N, (int)K,
                               ptr(dw), dt_of(dw, "fp8_linear"), ptr(db), dt_of(db, "fp8_linear"), ptr(work), n, stream_of(dy)),
                 "hcm_fp8_wgrad");
      } else {
        if (nw) dw.zero_();
        if (nb) db.zero_();
      }
    }
    return once({dx, dw, db, Tensor(), Tensor()});
  }
};

// `weight` (packed here, differentiable) or the four buffers of one that the caller keeps
Tensor fp8_linear(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& wq_, const OptTensor& ws_, const OptTensor& wqt_,
                  const OptTensor& wst_, at::IntArrayRef w_shape) {
  check_float(x, x, "fp8_linear");
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "fp8_linear: the last axis must have at least one element");
  const int64_t K = x.size(-1);
  const Tensor w = value(weight), b = value(bias);
  if (w.defined()) {
    check_float(w, x, "fp8_linear");
    w_shape = w.sizes();
  }
  TORCH_CHECK_VALUE(w_shape.size() == 2, "fp8_linear: a weight has two axes");
  check_width(K, w_shape[1], "fp8_linear");
  const int64_t N = w_shape[0];
  check_vector(b, x, N, "fp8_linear", "bias");
  TORCH_CHECK_VALUE(x.numel() / K <= INT32_MAX - 512, "fp8_linear: too many rows");
  check_no_tangent({&x, &w, &b}, "fp8_linear");
  const c10::DeviceGuard guard(x.device());
  Weight8 W;
  if (w.defined()) {
    at::AutoGradMode off(false);
    W = lay_out(w);
  } else {
    const Tensor wq = value(wq_), ws = value(ws_), wqt = value(wqt_), wst = value(wst_);
    TORCH_CHECK_VALUE(wq.defined() && ws.defined() && wqt.defined() && wst.defined(), "fp8_linear: no weight");
    check_weight(wq, ws, N, K, x, "fp8_linear");
    check_weight(wqt, wst, K, N, x, "fp8_linear");
    W = {wqt, wst, bytes(wq), bytes(ws), bytes(wqt), bytes(wst)};
  }
  if (!at::GradMode::is_enabled() || !(wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return linear_forward(rows_of(x, "fp8_linear"), W.q, W.scale, N, b, with_last(x.sizes(), N), nullptr);
  return Fp8Linear::apply(x, weight, bias, W, N);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(hcmoco, m) {
  m.def("act8_pack(Tensor x) -> (Tensor, Tensor)", &act8_pack);
  m.def("act8_unpack(Tensor q, Tensor scale, int[] shape, ScalarType dtype) -> Tensor", &act8_unpack);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool act8) -> Tensor", &layer_norm);
  m.def("fp8_weight(Tensor weight) -> (Tensor, Tensor, Tensor, Tensor)", &fp8_weight);
  m.def("fp8_matmul(Tensor q, Tensor scale, int[] shape, Tensor wq, Tensor ws, int[] w_shape, Tensor? bias, ScalarType dtype) -> Tensor", &fp8_matmul);
  m.def("fp8_linear(Tensor x, Tensor? weight, Tensor? bias, Tensor? wq, Tensor? ws, Tensor? wqt, Tensor? wst, int[] w_shape) -> Tensor", &fp8_linear);
}
