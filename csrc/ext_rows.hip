// Torch bindings of the row operators: layer_norm and linear_act.
#include <torch/extension.h>

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include "rows.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

#define DISPATCH_FT(dtype, ...)                            \
  do {                                                     \
    if ((dtype) == torch::kFloat32) {                      \
      using scalar_t = float;                              \
      __VA_ARGS__;                                         \
    } else {                                               \
      using scalar_t = gfa::bf16;                          \
      __VA_ARGS__;                                         \
    }                                                      \
  } while (0)

hipStream_t cur_stream() {
  return c10::hip::getCurrentHIPStream().stream();
}

void check(const Tensor& t, const Tensor& x, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), what,
              ": on another device than x");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 ||
                  t.scalar_type() == torch::kBFloat16,
              what, ": expected float32 or bfloat16, got ", t.scalar_type());
}

void check_param(const OptTensor& p, const Tensor& x, int64_t n,
                 const char* what) {
  if (!p) return;
  check(*p, x, what);
  TORCH_CHECK(p->dim() == 1 && p->size(0) == n, what, ": expected [", n, "]");
  TORCH_CHECK(p->scalar_type() == x.scalar_type() ||
                  p->scalar_type() == torch::kFloat32,
              what, ": expected x's dtype or float32");
}

// A tensor [..., n] as rows of n contiguous elements at one stride
struct Rows {
  Tensor t;  // what is read: the tensor itself or a contiguous copy
  int64_t count, stride;
};

Rows rows_of(const Tensor& t) {
  const int64_t n = t.size(-1);
  Rows r{t, 1, n};
  bool ok = t.stride(-1) == 1 || n == 1;
  bool first = true;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    const int64_t size = t.size(d), stride = t.stride(d);
    if (size != 1) {
      if (first) {
        r.stride = stride;
        first = false;
      } else if (stride != r.stride * r.count) {
        ok = false;
      }
    }
    r.count *= size;
  }
  if (!ok) {
    r.t = t.contiguous();
    r.stride = n;
  }
  return r;
}

template <typename T>
const T* cptr(const Tensor& t) {
  return static_cast<const T*>(t.data_ptr());
}
template <typename T>
const T* cptr(const OptTensor& t) {
  return t ? static_cast<const T*>(t->data_ptr()) : nullptr;
}
template <typename T>
T* mptr(const OptTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// ---- layer norm ----

// calls f(T, P) for the types of x and of the parameters
#define DISPATCH_TP(x, p32, ...)                               \
  do {                                                         \
    if ((x).scalar_type() == torch::kFloat32) {                \
      using T = float;                                         \
      using P = float;                                         \
      __VA_ARGS__;                                             \
    } else if (p32) {                                          \
      using T = gfa::bf16;                                     \
      using P = float;                                         \
      __VA_ARGS__;                                             \
    } else {                                                   \
      using T = gfa::bf16;                                     \
      using P = gfa::bf16;                                     \
      __VA_ARGS__;                                             \
    }                                                          \
  } while (0)

bool params_f32(const OptTensor& w, const OptTensor& b) {
  TORCH_CHECK(!w || !b || w->scalar_type() == b->scalar_type(),
              "layer_norm: weight and bias differ in dtype");
  return w ? w->scalar_type() == torch::kFloat32
           : !b || b->scalar_type() == torch::kFloat32;
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_fwd(
    const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
    bool save) {
  check(x, x, "layer_norm: x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1 << 30),
              "layer_norm: size of the last dimension");
  const int n = (int)x.size(-1);
  check_param(w, x, n, "layer_norm: weight");
  check_param(b, x, n, "layer_norm: bias");
  const bool p32 = params_f32(w, b);
  c10::hip::HIPGuard guard(x.get_device());
  const OptTensor wc = w ? OptTensor(w->contiguous()) : w;
  const OptTensor bc = b ? OptTensor(b->contiguous()) : b;
  const Rows xr = rows_of(x);
  Tensor y = torch::empty(x.sizes(), x.options());
  OptTensor mean, rstd;
  if (save) {
    mean = torch::empty({xr.count}, x.options().dtype(torch::kFloat32));
    rstd = torch::empty({xr.count}, x.options().dtype(torch::kFloat32));
  }
  if (xr.count > 0) {
    DISPATCH_TP(x, p32, {
      gfa::launch_layer_norm_fwd<T, P>(
          static_cast<T*>(y.data_ptr()), mptr<float>(mean), mptr<float>(rstd),
          cptr<T>(xr.t), xr.stride, cptr<P>(wc), cptr<P>(bc), xr.count, n,
          (float)eps, cur_stream());
    });
    HIP_CHECK_LAST();
  }
  return {y, mean, rstd};
}

std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_bwd(
    const Tensor& dy, const Tensor& x, const OptTensor& w, const OptTensor& b,
    const Tensor& mean, const Tensor& rstd, bool need_dx, bool need_dw,
    bool need_db) {
  check(x, x, "layer_norm: x");
  check(dy, x, "layer_norm: dy");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1 << 30),
              "layer_norm: size of the last dimension");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(),
              "layer_norm: dy does not fit x");
  const int n = (int)x.size(-1);
  check_param(w, x, n, "layer_norm: weight");
  check_param(b, x, n, "layer_norm: bias");
  const bool p32 = params_f32(w, b);
  c10::hip::HIPGuard guard(x.get_device());
  const OptTensor wc = w ? OptTensor(w->contiguous()) : w;
  const Rows xr = rows_of(x), dr = rows_of(dy);
  for (const Tensor& s : {mean, rstd})
    TORCH_CHECK(s.device() == x.device() && s.is_contiguous() &&
                    s.scalar_type() == torch::kFloat32 &&
                    s.numel() == xr.count,
                "layer_norm: statistics do not fit x");
  const auto f32 = x.options().dtype(torch::kFloat32);
  const auto popt = p32 ? f32 : x.options();
  OptTensor dx, dw, db, partial;
  if (need_dx) dx = torch::empty(x.sizes(), x.options());
  if (xr.count == 0) {
    if (need_dw) dw = torch::zeros({n}, popt);
    if (need_db) db = torch::zeros({n}, popt);
    return {dx, dw, db};
  }
  if (need_dw) dw = torch::empty({n}, popt);
  if (need_db) db = torch::empty({n}, popt);
  if (need_dw || need_db)
    partial = torch::empty({2, gfa::layer_norm_bwd_groups(
                                   xr.count, n,
                                   x.scalar_type() == torch::kFloat32),
                            n},
                           f32);
  DISPATCH_TP(x, p32, {
    gfa::launch_layer_norm_bwd<T, P>(
        mptr<T>(dx), mptr<P>(dw), mptr<P>(db), mptr<float>(partial),
        cptr<T>(dr.t), dr.stride, cptr<T>(xr.t), xr.stride, cptr<P>(wc),
        cptr<float>(mean), cptr<float>(rstd), xr.count, n, cur_stream());
  });
  HIP_CHECK_LAST();
  return {dx, dw, db};
}

// ---- linear ----

void check_linear(const Tensor& x, const Tensor& w, const OptTensor& bias) {
  check(x, x, "linear_act: x");
  check(w, x, "linear_act: weight");
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1) &&
                  w.size(0) >= 1 && w.size(1) >= 1 &&
                  w.size(0) <= (1 << 22) && w.size(1) <= (1 << 22) &&
                  w.scalar_type() == x.scalar_type(),
              "linear_act: weight does not fit x");
  check_param(bias, x, w.size(0), "linear_act: bias");
}

std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}

std::tuple<Tensor, OptTensor> linear_act_fwd(
    const Tensor& x, const Tensor& w, const OptTensor& bias,
    const OptTensor& residual, int64_t act, double alpha, double gain,
    double clamp, double weight_gain, double bias_gain, bool save_z) {
  check_linear(x, w, bias);
  TORCH_CHECK(act >= 0 && act <= gfa::kSilu, "linear_act: activation");
  const int64_t n = w.size(0), k = w.size(1);
  const auto shape = out_shape(x, n);
  if (residual) {
    check(*residual, x, "linear_act: residual");
    TORCH_CHECK(residual->sizes() == shape &&
                    residual->scalar_type() == x.scalar_type(),
                "linear_act: residual does not fit");
  }
  c10::hip::HIPGuard guard(x.get_device());
  const Rows xr = rows_of(x), wr = rows_of(w);
  const OptTensor bc = bias ? OptTensor(bias->contiguous()) : bias;
  Tensor y = torch::empty(shape, x.options());
  OptTensor z;
  if (save_z) z = torch::empty(shape, x.options());
  if (xr.count == 0) return {y, z};
  const gfa::GemmArgs g{xr.count, n,         k, xr.stride, 1,
                        wr.stride, 1, (float)weight_gain};
  DISPATCH_FT(x.scalar_type(), {
    gfa::EpilogueArgs<scalar_t> e{};
    if (bc) {
      e.bias = bc->data_ptr();
      e.bias_f32 = bc->scalar_type() == torch::kFloat32;
      e.bias_gain = (float)bias_gain;
    }
    Rows rr;
    if (residual) {
      rr = rows_of(*residual);
      e.residual = cptr<scalar_t>(rr.t);
      e.res_stride = rr.stride;
    }
    e.z = mptr<scalar_t>(z);
    e.act = {(int)act, (float)alpha, (float)gain, (float)clamp};
    gfa::launch_linear_gemm<scalar_t>(static_cast<scalar_t*>(y.data_ptr()),
                                      cptr<scalar_t>(xr.t),
                                      cptr<scalar_t>(wr.t), g, e,
                                      cur_stream());
  });
  HIP_CHECK_LAST();
  return {y, z};
}

std::tuple<OptTensor, OptTensor, OptTensor> linear_act_bwd(
    const Tensor& dy, const OptTensor& z, const Tensor& x, const Tensor& w,
    const OptTensor& bias, int64_t act, double alpha, double gain,
    double clamp, double weight_gain, double bias_gain, bool need_dx,
    bool need_dw, bool need_db) {
  check_linear(x, w, bias);
  TORCH_CHECK(act >= 0 && act <= gfa::kSilu, "linear_act: activation");
  const int64_t n = w.size(0), k = w.size(1);
  const auto shape = out_shape(x, n);
  check(dy, x, "linear_act: dy");
  TORCH_CHECK(dy.sizes() == shape && dy.scalar_type() == x.scalar_type(),
              "linear_act: dy does not fit");
  TORCH_CHECK(!need_db || bias, "linear_act: no bias");
  TORCH_CHECK(z || (act == gfa::kLinear && std::isinf(clamp)),
              "linear_act: the pre-activation is missing");
  if (z)
    TORCH_CHECK(z->device() == x.device() && z->is_contiguous() &&
                    z->sizes() == shape &&
                    z->scalar_type() == x.scalar_type(),
                "linear_act: z does not fit");
  c10::hip::HIPGuard guard(x.get_device());
  const Rows xr = rows_of(x), wr = rows_of(w), dr = rows_of(dy);
  const int64_t m = xr.count;
  OptTensor dx, dw, db, dz, partial;
  if (need_dx) dx = torch::empty(x.sizes(), x.options());
  if (m == 0) {
    if (need_dw) dw = torch::zeros(w.sizes(), w.options());
    if (need_db) db = torch::zeros({n}, bias->options());
    return {dx, dw, db};
  }
  if (need_dw) dw = torch::empty(w.sizes(), w.options());
  if (need_db) db = torch::empty({n}, bias->options());
  // without z the slope is the gain everywhere: dz is dy and the products
  // carry the factor
  const double slope = z ? 1.0 : gain;
  const int groups = gfa::linear_dz_groups(m, (int)n);
  if (!need_dx && !need_dw && !need_db) return {dx, dw, db};
  if (z) dz = torch::empty(shape, x.options());
  if (need_db)
    partial =
        torch::empty({groups, n}, x.options().dtype(torch::kFloat32));
  DISPATCH_FT(x.scalar_type(), {
    const gfa::ActParams ap{(int)act, (float)alpha, (float)gain,
                            (float)clamp};
    if (z || need_db)
      gfa::launch_linear_dz<scalar_t>(
          mptr<scalar_t>(dz), mptr<float>(partial), cptr<scalar_t>(dr.t),
          dr.stride, cptr<scalar_t>(z), ap, m, (int)n, cur_stream());
    if (need_db) {
      const float scale = (float)(bias_gain * slope);
      if (bias->scalar_type() == torch::kFloat32)
        gfa::launch_sum_groups<float>(mptr<float>(db), nullptr,
                                      partial->data_ptr<float>(), groups,
                                      (int)n, scale, cur_stream());
      else
        gfa::launch_sum_groups<gfa::bf16>(mptr<gfa::bf16>(db), nullptr,
                                          partial->data_ptr<float>(), groups,
                                          (int)n, scale, cur_stream());
    }
    const scalar_t* d = z ? cptr<scalar_t>(dz) : cptr<scalar_t>(dr.t);
    const int64_t ds = z ? n : dr.stride;
    gfa::EpilogueArgs<scalar_t> e{};
    e.act = {gfa::kLinear, 0.f, 1.f, INFINITY};
    const float scale = (float)(weight_gain * slope);
    if (need_dx)
      gfa::launch_linear_gemm<scalar_t>(
          mptr<scalar_t>(dx), d, cptr<scalar_t>(wr.t),
          {m, k, n, ds, 1, 1, wr.stride, scale}, e, cur_stream());
    if (need_dw)
      gfa::launch_linear_gemm<scalar_t>(
          mptr<scalar_t>(dw), d, cptr<scalar_t>(xr.t),
          {n, k, m, 1, ds, 1, xr.stride, scale}, e, cur_stream());
  });
  HIP_CHECK_LAST();
  return {dx, dw, db};
}

}  // namespace

void bind_rows(pybind11::module& m) {
  m.def("layer_norm_fwd", &layer_norm_fwd,
        "layer norm -> (y, mean, rstd)");
  m.def("layer_norm_bwd", &layer_norm_bwd, "layer norm -> (dx, dw, db)");
  m.def("linear_act_fwd", &linear_act_fwd,
        "clamp(act(x W^T + b) * gain) + residual -> (y, z)");
  m.def("linear_act_bwd", &linear_act_bwd, "linear_act -> (dx, dW, db)");
}
