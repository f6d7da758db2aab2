// The torch side of the token operators (gs3d_b200/rotary.py, norm.py, attention.py): checks of
// arguments, outputs and workspaces, and the autograd functions around the C entry points of
// include/gs3d_b200.h. It is native because these calls are short: through ctypes and Python
// autograd functions the host took 26 us for a rotary call of 3 us and 155 us for a norm's forward
// and backward of 36 us. The entry points' addresses come from the library that
// custom_rasterizer_cuda._lib has loaded (bind).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <array>
#include <cmath>
#include <string>

#include "gs3d_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

struct Entry {
  decltype(&gs_last_error) last_error = nullptr;
  decltype(&gs_rotary_axes) rotary_axes = nullptr;
  decltype(&gs_rms_norm_forward) rms_norm_forward = nullptr;
  decltype(&gs_rms_norm_e4m3) rms_norm_e4m3 = nullptr;
  decltype(&gs_rms_norm_backward_workspace_size) rms_norm_backward_workspace_size = nullptr;
  decltype(&gs_rms_norm_backward) rms_norm_backward = nullptr;
  decltype(&gs_cross_attention_workspace_size) cross_attention_workspace_size = nullptr;
  decltype(&gs_cross_attention_forward) cross_attention_forward = nullptr;
  decltype(&gs_cross_attention_backward_workspace_size) cross_attention_backward_workspace_size =
      nullptr;
  decltype(&gs_cross_attention_backward) cross_attention_backward = nullptr;
} entry;

template <typename F>
void bind_one(const py::dict& addresses, const char* name, F& f) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& addresses) {
#define GS_BIND(name) bind_one(addresses, "gs_" #name, entry.name)
  GS_BIND(last_error);
  GS_BIND(rotary_axes);
  GS_BIND(rms_norm_forward);
  GS_BIND(rms_norm_e4m3);
  GS_BIND(rms_norm_backward_workspace_size);
  GS_BIND(rms_norm_backward);
  GS_BIND(cross_attention_workspace_size);
  GS_BIND(cross_attention_forward);
  GS_BIND(cross_attention_backward_workspace_size);
  GS_BIND(cross_attention_backward);
#undef GS_BIND
}

void check(int status) {
  if (status != GS_OK)
    throw std::runtime_error("gs3d_b200 error " + std::to_string(status) + ": " +
                             entry.last_error());
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GS_FP32;
    case at::kHalf: return GS_FP16;
    case at::kBFloat16: return GS_BF16;
    default: return -1;
  }
}

void check_tokens(const Tensor& t, const char* name, int64_t dims) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions");
}

// What is told apart by neither requires_grad() nor the pointers: a trace would record the empty
// output and not the kernel, and a tangent (forward mode) would be dropped without a word.
void check_untraced(const char* op) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), op, " cannot be traced");
}

bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

void check_no_tangent(const char* op, std::initializer_list<const Tensor*> inputs) {
  check_untraced(op);
  for (const Tensor* t : inputs)
    TORCH_CHECK(!has_tangent(*t), op, " has no forward-mode derivative");
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void* data_of(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
void* data_of(const OptTensor& t) { return t ? data_of(*t) : nullptr; }

// t, or a contiguous copy of it where its last axis is not contiguous, where its address or strides
// are not multiples of `elements` elements (those of axes of length 1 do not count), or, with
// `elements` above 1, where an axis other than the first repeats itself (a stride of 0).
Tensor usable(const Tensor& t, int64_t elements) {
  if (t.numel() == 0) return t;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % (elements * t.element_size()))
    return t.clone(at::MemoryFormat::Contiguous);
  const int64_t last = t.dim() - 1;
  bool fine = t.stride(last) == 1 || t.size(last) == 1;
  for (int64_t i = 0; i < last && fine; ++i)
    if (t.size(i) > 1)
      fine = t.stride(i) % elements == 0 && (elements == 1 || i == 0 || t.stride(i) != 0);
  return fine ? t : t.contiguous();
}

gs_token_view view4(const Tensor& t) {
  const auto stride = [&](int64_t i) { return (long long)(t.size(i) > 1 ? t.stride(i) : 0); };
  return {data_of(t), stride(0), stride(1), stride(2)};
}

// ---- rotary positions ------------------------------------------------------------------------
struct RotaryArgs {
  int n = 0;
  std::array<int, 4> dims{};
  std::array<double, 4> bases{};
  bool interleaved = false, inverse = false;
};

Tensor rotate(const Tensor& x_in, const Tensor& positions, const RotaryArgs& a) {
  const Tensor x = usable(x_in, 1);
  const Tensor y = at::empty(x.sizes(), x.options());
  if (y.numel() == 0) return y;
  const gs_token_view xv = view4(x), yv = view4(y);
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  check(entry.rotary_axes(type_of(x), (int)x.size(0), (int)x.size(1), (int)x.size(2),
                          (int)x.size(3), &xv, &yv, positions.data_ptr(),
                          positions.scalar_type() == at::kInt ? GS_INT32 : GS_FP32,
                          positions.size(0) > 1 ? positions.stride(0) : 0, positions.stride(1),
                          a.n, a.dims.data(), a.bases.data(), a.interleaved, a.inverse,
                          stream_of(x)));
  return y;
}

Tensor differentiable_rotate(const Tensor& x, const Tensor& positions, const RotaryArgs& a);

struct RotaryAxes : torch::autograd::Function<RotaryAxes> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions,
                        const RotaryArgs& a) {
    ctx->save_for_backward({positions});
    ctx->saved_data["ints"] = std::vector<int64_t>{a.n,       a.dims[0], a.dims[1],    a.dims[2],
                                                   a.dims[3], a.inverse, a.interleaved};
    ctx->saved_data["bases"] = std::vector<double>(a.bases.begin(), a.bases.end());
    return rotate(x, positions, a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor positions = ctx->get_saved_variables()[0];
    const auto ints = ctx->saved_data["ints"].toIntVector();
    const auto bases = ctx->saved_data["bases"].toDoubleVector();
    RotaryArgs a;
    a.n = (int)ints[0];
    for (int i = 0; i < 4; ++i) a.dims[i] = (int)ints[1 + i], a.bases[i] = bases[i];
    a.inverse = !ints[5];
    a.interleaved = ints[6];
    return {differentiable_rotate(grads[0], positions, a), Tensor(), Tensor()};
  }
};

// The map is linear: its gradient, a second derivative and the tangent (forward mode) are rotations.
Tensor differentiable_rotate(const Tensor& x, const Tensor& positions, const RotaryArgs& a) {
  if (has_tangent(x)) {
    const auto [value, tangent] = at::_unpack_dual(x, /*level=*/0);
    return at::_make_dual(differentiable_rotate(value, positions, a),
                          differentiable_rotate(tangent, positions, a), /*level=*/0);
  }
  return x.requires_grad() && at::GradMode::is_enabled()
             ? RotaryAxes::apply(x, positions.detach(), a)
             : rotate(x, positions, a);
}

Tensor rotary_axes(const Tensor& x, Tensor positions, const std::vector<int64_t>& axis_dims,
                   const std::vector<double>& bases, bool interleaved, bool inverse) {
  check_untraced("rotary_axes");
  check_tokens(x, "x", 4);
  check_tokens(positions, "positions", 3);
  TORCH_CHECK(type_of(x) >= 0, "x must be float32, float16 or bfloat16");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kFloat,
              "positions must be int32 or float32");
  TORCH_CHECK(positions.device() == x.device(), "x and positions must be on the same device");
  const int64_t n = (int64_t)axis_dims.size(), D = x.size(3);
  TORCH_CHECK(n >= 1 && n <= 4, "between 1 and 4 axes");
  TORCH_CHECK((positions.size(0) == 1 || positions.size(0) == x.size(0)) &&
                  positions.size(1) == x.size(1) && positions.size(2) == n,
              "positions must be [B or 1, L, number of axes]");
  TORCH_CHECK(D % 2 == 0 && D >= 2 && D <= 256, "the head size must be even, between 2 and 256");
  RotaryArgs a;
  a.n = (int)n;
  a.interleaved = interleaved;
  a.inverse = inverse;
  int64_t sum = 0;
  bool fine = true;
  for (int64_t i = 0; i < n; ++i) {
    fine = fine && axis_dims[i] >= 2 && axis_dims[i] <= D && axis_dims[i] % 2 == 0;
    sum += axis_dims[i];
    a.dims[i] = (int)axis_dims[i];
  }
  TORCH_CHECK(fine && sum <= D,
              "axis_dims must be even, at least 2, and add up to at most the head size");
  fine = (int64_t)bases.size() == n;
  for (int64_t i = 0; i < n && fine; ++i) {
    a.bases[i] = bases[i];
    fine = a.bases[i] > 0 && std::isfinite(a.bases[i]);
  }
  TORCH_CHECK(fine, "base must be one positive number, or one for each axis");
  if (positions.stride(2) != 1) positions = positions.contiguous();
  return differentiable_rotate(x, positions, a);
}

// ---- norms -----------------------------------------------------------------------------------
constexpr int64_t kMaxWidth = 32768;

void check_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps) {
  const auto one = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.scalar_type() == x.scalar_type() && t.device() == x.device(), name,
                " must have x's type and device");
  };
  one(x, "x");
  one(weight, "weight");
  if (residual) one(*residual, "residual");
  TORCH_CHECK(type_of(x) >= 0, "x must be float32, float16 or bfloat16");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxWidth,
              "the last axis must have between 1 and ", kMaxWidth, " elements");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1),
              "weight must have one element for each of the last axis");
  TORCH_CHECK(!residual || residual->sizes() == x.sizes(), "residual must have x's shape");
  TORCH_CHECK(eps >= 0.0, "eps must be non-negative");
}

struct NormOut {
  Tensor y, h, rstd;
};

// x, weight and residual contiguous
NormOut norm_forward(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps,
                     bool save) {
  const int64_t width = x.size(-1), rows = x.numel() / width;
  NormOut o;
  o.y = at::empty_like(x);
  if (residual) o.h = at::empty_like(x);
  if (save) o.rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (rows) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    check(entry.rms_norm_forward(type_of(x), rows, (int)width, x.data_ptr(), data_of(residual),
                                 weight.data_ptr(), (float)eps, o.y.data_ptr(),
                                 residual ? o.h.data_ptr() : nullptr,
                                 save ? static_cast<float*>(o.rstd.data_ptr()) : nullptr,
                                 stream_of(x)));
  }
  return o;
}

std::pair<Tensor, Tensor> norm_backward(Tensor dy, const Tensor& dh_in, const Tensor& h,
                                        const Tensor& weight, const Tensor& rstd) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm has no second derivative");
  check_no_tangent("rms_norm's gradient", {&dy, dh_in.defined() ? &dh_in : &dy});
  const int64_t width = h.size(-1), rows = h.numel() / width;
  dy = dy.contiguous();
  const Tensor dh = dh_in.defined() ? dh_in.contiguous() : dh_in;
  const Tensor dx = at::empty_like(h), dw = at::empty_like(weight);
  const c10::cuda::OptionalCUDAGuard guard(h.device());
  const size_t bytes = entry.rms_norm_backward_workspace_size(rows, (int)width);
  const Tensor ws = at::empty({(int64_t)bytes}, h.options().dtype(at::kByte));
  check(entry.rms_norm_backward(type_of(h), rows, (int)width, data_of(dy),
                                dh.defined() ? data_of(dh) : nullptr, data_of(h),
                                weight.data_ptr(), static_cast<const float*>(data_of(rstd)),
                                data_of(dx), dw.data_ptr(), data_of(ws), bytes, stream_of(h)));
  return {dx, dw};
}

struct RMSNorm : torch::autograd::Function<RMSNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, double eps) {
    const NormOut o = norm_forward(x, weight, c10::nullopt, eps, true);
    ctx->save_for_backward({x, weight, o.rstd});
    return o.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = norm_backward(grads[0], Tensor(), saved[0], saved[1], saved[2]);
    return {dx, dw, Tensor()};
  }
};

struct RMSNormResidual : torch::autograd::Function<RMSNormResidual> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               const Tensor& residual, double eps) {
    ctx->set_materialize_grads(false);
    const NormOut o = norm_forward(x, weight, residual, eps, true);
    ctx->save_for_backward({o.h, weight, o.rstd});
    return {o.y, o.h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined())  // only the residual stream was used
      return {grads[1], Tensor(), grads[1], Tensor()};
    const auto saved = ctx->get_saved_variables();
    auto [dx, dw] = norm_backward(grads[0], grads[1], saved[0], saved[1], saved[2]);
    return {dx, dw, dx, Tensor()};
  }
};

py::object rms_norm(Tensor x, Tensor weight, OptTensor residual, double eps) {
  check_no_tangent("rms_norm", {&x, &weight, residual ? &*residual : &x});
  check_norm(x, weight, residual, eps);
  Tensor y, h;
  {
    py::gil_scoped_release release;
    x = x.contiguous();
    weight = weight.contiguous();
    if (residual) residual = residual->contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() ||
                                       (residual && residual->requires_grad()))) {
      if (residual) {
        const auto out = RMSNormResidual::apply(x, weight, *residual, eps);
        y = out[0], h = out[1];
      } else {
        y = RMSNorm::apply(x, weight, eps);
      }
    } else {
      const NormOut o = norm_forward(x, weight, residual, eps, false);
      y = o.y, h = o.h;
    }
  }
  return residual ? py::cast(std::make_tuple(y, h)) : py::cast(y);
}

py::object rms_norm_8bit(Tensor x, Tensor weight, OptTensor residual, double eps, int64_t group) {
  check_no_tangent("rms_norm_8bit", {&x, &weight, residual ? &*residual : &x});
  check_norm(x, weight, residual, eps);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(x.requires_grad() || weight.requires_grad() ||
                                               (residual && residual->requires_grad())),
              "rms_norm_8bit has no gradient");
  const int64_t width = x.size(-1);
  TORCH_CHECK(group == 0 || (group == 128 && width % 128 == 0),
              "group must be 0 (one scale a row) or 128, dividing the width");
  x = x.contiguous();
  weight = weight.contiguous();
  if (residual) residual = residual->contiguous();
  if (group) {  // read 16 bytes at a time
    const int64_t per = 16 / x.element_size();
    x = usable(x, per);
    weight = usable(weight, per);
    if (residual) residual = usable(*residual, per);
  }
  const int64_t rows = x.numel() / width;
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = group ? width / group : 1;
  const Tensor scales = at::empty(shape, x.options().dtype(at::kFloat));
  Tensor h;
  if (residual) h = at::empty_like(x);
  if (rows) {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    check(entry.rms_norm_e4m3(type_of(x), rows, (int)width, (int)group, x.data_ptr(),
                              data_of(residual), weight.data_ptr(), (float)eps, q.data_ptr(),
                              static_cast<float*>(scales.data_ptr()),
                              residual ? h.data_ptr() : nullptr, stream_of(x)));
  }
  return residual ? py::cast(std::make_tuple(q, scales, h)) : py::cast(std::make_tuple(q, scales));
}

// ---- cross attention ---------------------------------------------------------------------------
gs_attention_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const OptTensor& lengths, const OptTensor& mask, double scale,
                                 const Tensor& out, const Tensor& lse) {
  gs_attention_args a{};
  a.dtype = type_of(q);
  a.B = (int)q.size(0), a.Lq = (int)q.size(1), a.Hq = (int)q.size(2), a.D = (int)q.size(3);
  a.Lk = (int)k.size(1), a.Hkv = (int)k.size(2);
  a.scale = (float)scale;
  a.q = view4(q), a.k = view4(k), a.v = view4(v), a.out = view4(out);
  a.lengths = static_cast<const int*>(data_of(lengths));
  if (mask && mask->numel()) {
    a.mask = static_cast<const unsigned char*>(mask->data_ptr());
    const auto stride = [&](int64_t i) {
      return (long long)(mask->size(i) > 1 ? mask->stride(i) : 0);
    };
    a.mask_batch_stride = stride(0);
    a.mask_head_stride = stride(1);
    a.mask_query_stride = stride(2);
  }
  a.lse = lse.defined() ? static_cast<float*>(data_of(lse)) : nullptr;
  return a;
}

std::pair<Tensor, Tensor> attend(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const OptTensor& lengths, const OptTensor& mask, double scale,
                                 bool want_lse) {
  const Tensor out = at::empty(q.sizes(), q.options());
  Tensor lse;
  if (want_lse)
    lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  if (out.numel() == 0) return {out, lse};
  const gs_attention_args a = attention_args(q, k, v, lengths, mask, scale, out, lse);
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const size_t bytes = entry.cross_attention_workspace_size(&a);
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  check(entry.cross_attention_forward(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)));
  return {out, lse};
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k,
                               const Tensor& v, const OptTensor& lengths, const OptTensor& mask,
                               double scale) {
    ctx->set_materialize_grads(false);
    auto [out, lse] = attend(q, k, v, lengths, mask, scale, true);
    ctx->save_for_backward({q, k, v, out, lse, lengths.value_or(Tensor()), mask.value_or(Tensor())});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    TORCH_CHECK(!at::GradMode::is_enabled(), "cross_attention has no second derivative");
    check_no_tangent("cross_attention's gradient", {&grads[0]});
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    const auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; };
    const Tensor dout = usable(grads[0], 8);
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                 dv = at::empty(v.sizes(), v.options());
    const gs_attention_args a = attention_args(q, k, v, given(saved[5]), given(saved[6]),
                                               ctx->saved_data["scale"].toDouble(), out, lse);
    const gs_token_view views[4] = {view4(dout), view4(dq), view4(dk), view4(dv)};
    const c10::cuda::OptionalCUDAGuard guard(q.device());
    const size_t bytes = entry.cross_attention_backward_workspace_size(&a);
    const Tensor ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    check(entry.cross_attention_backward(&a, &views[0], &views[1], &views[2], &views[3],
                                         data_of(ws), bytes, stream_of(q)));
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};

py::object cross_attention(Tensor q, Tensor k, Tensor v, OptTensor lengths, OptTensor mask,
                           c10::optional<double> scale_in, bool return_lse) {
  check_no_tangent("cross_attention", {&q, &k, &v});
  check_tokens(q, "q", 4);
  check_tokens(k, "k", 4);
  check_tokens(v, "v", 4);
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "q must be float16 or bfloat16");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "q, k and v must have the same type");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device(),
              "q, k and v must be on one device");
  const int64_t B = q.size(0), Lq = q.size(1), Hq = q.size(2), D = q.size(3), Lk = k.size(1),
                Hkv = k.size(2);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D,
              "k and v must be [B, Lk, Hkv, D] with q's B and D");
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "the head size must be a multiple of 8 up to 128");
  TORCH_CHECK(Hkv == 0 ? Hq == 0 : Hq % Hkv == 0, "the key heads must divide the query heads");
  TORCH_CHECK(B < (1ll << 31) && Lq < (1ll << 31) && Lk < (1ll << 31) && Hq < (1ll << 31),
              "sizes must be below 2^31");
  if (lengths) {
    TORCH_CHECK(lengths->device() == q.device() && lengths->scalar_type() == at::kInt &&
                    lengths->dim() == 1 && lengths->size(0) == B,
                "lengths must be an int32 tensor [B] on q's device");
    lengths = lengths->contiguous();
  }
  if (mask) {
    TORCH_CHECK(mask->device() == q.device() && mask->scalar_type() == at::kBool &&
                    mask->dim() == 4,
                "mask must be a bool tensor of 4 dimensions on q's device");
    const auto either = [&](int64_t i, int64_t n) { return mask->size(i) == 1 || mask->size(i) == n; };
    TORCH_CHECK(either(0, B) && either(1, Hq) && either(2, Lq) && mask->size(3) == Lk,
                "mask must be [B or 1, Hq or 1, Lq or 1, Lk]");
    if (Lk > 1 && mask->stride(3) != 1) mask = mask->contiguous();
  }
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)D);
  TORCH_CHECK(std::isfinite(scale), "scale must be finite");
  Tensor out, lse;
  {
    py::gil_scoped_release release;
    q = usable(q, 8);
    k = usable(k, 8);
    v = usable(v, 8);
    if (at::GradMode::is_enabled() &&
        (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      const auto o = CrossAttention::apply(q, k, v, lengths, mask, scale);
      out = o[0], lse = o[1];
    } else {
      std::tie(out, lse) = attend(q, k, v, lengths, mask, scale, return_lse);
    }
  }
  return return_lse ? py::cast(std::make_tuple(out, lse)) : py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("bind", &bind);
  m.def("rotary_axes", &rotary_axes, py::call_guard<py::gil_scoped_release>());
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_8bit", &rms_norm_8bit);
  m.def("cross_attention", &cross_attention);
}
