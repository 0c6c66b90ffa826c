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
                  w.size(0) < (1 << 20) && w.size(1) < (1 << 20) &&
                  w.scalar_type() == x.scalar_type(),
              "linear_act: weight does not fit x");
  check_param(bias, x, w.size(0), "linear_act: bias");
}

std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}

// The tiles read rows of 16-byte granules: rows elsewhere, or of another
// width, are copied to padded ones (zeros behind the last element).
template <typename T>
Rows tile_rows(const Rows& r, int64_t n) {
  const int64_t v = 16 / sizeof(T);
  const int64_t width = (n + 7) / 8 * 8;
  if (n % v == 0 && r.stride % v == 0 && r.stride < (1 << 20) &&
      reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16 == 0)
    return r;
  Rows p{torch::empty({r.count, width}, r.t.options()), r.count, width};
  gfa::launch_pad_rows<T>(static_cast<T*>(p.t.data_ptr()), cptr<T>(r.t),
                          r.stride, r.count, (int)n, (int)width, cur_stream());
  return p;
}

template <typename T>
gfa::EpilogueArgs<T> epilogue(const OptTensor& bias, int64_t act, double alpha,
                              double gain, double clamp, double bias_gain) {
  gfa::EpilogueArgs<T> e{};
  if (bias) {
    e.bias = bias->data_ptr();
    e.bias_f32 = bias->scalar_type() == torch::kFloat32;
    e.bias_gain = (float)bias_gain;
  }
  e.act = {(int)act, (float)alpha, (float)gain, (float)clamp};
  return e;
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
  const OptTensor bc = bias ? OptTensor(bias->contiguous()) : bias;
  Tensor y = torch::empty(shape, x.options());
  OptTensor z;
  if (save_z) z = torch::empty(shape, x.options().dtype(torch::kFloat32));
  if (y.numel() == 0) return {y, z};
  DISPATCH_FT(x.scalar_type(), {
    const Rows xr = tile_rows<scalar_t>(rows_of(x), k);
    const Rows wr = tile_rows<scalar_t>(rows_of(w), k);
    auto e = epilogue<scalar_t>(bc, act, alpha, gain, clamp, bias_gain);
    Rows rr;
    if (residual) {
      rr = rows_of(*residual);
      e.residual = cptr<scalar_t>(rr.t);
      e.res_stride = rr.stride;
    }
    e.z = mptr<float>(z);
    gfa::launch_linear_forward<scalar_t>(
        static_cast<scalar_t*>(y.data_ptr()), cptr<scalar_t>(xr.t),
        cptr<scalar_t>(wr.t),
        {xr.count, n, k, xr.stride, wr.stride, n, (float)weight_gain, k}, e,
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
  if (z)
    TORCH_CHECK(z->device() == x.device() && z->is_contiguous() &&
                    z->sizes() == shape &&
                    z->scalar_type() == torch::kFloat32,
                "linear_act: z does not fit");
  c10::hip::HIPGuard guard(x.get_device());
  const int64_t m = dy.numel() / n;
  OptTensor dx, dw, db;
  if (need_dx) dx = torch::empty(x.sizes(), x.options());
  if (m == 0) {
    if (need_dw) dw = torch::zeros(w.sizes(), w.options());
    if (need_db) db = torch::zeros({n}, bias->options());
    return {dx, dw, db};
  }
  if (need_dw) dw = torch::empty(w.sizes(), w.options());
  if (need_db) db = torch::empty({n}, bias->options());
  if (!need_dx && !need_dw && !need_db) return {dx, dw, db};
  const OptTensor bc = bias ? OptTensor(bias->contiguous()) : bias;
  const auto f32 = x.options().dtype(torch::kFloat32);
  // Without an activation or a clamp the slope is the gain everywhere: dz is
  // dy and the products carry the factor.
  const bool curved = act != gfa::kLinear || !std::isinf(clamp);
  const double slope = curved ? 1.0 : gain;
  DISPATCH_FT(x.scalar_type(), {
    const Rows xr = tile_rows<scalar_t>(rows_of(x), k);
    const Rows wr = tile_rows<scalar_t>(rows_of(w), k);
    Rows dr = rows_of(dy);
    auto e = epilogue<scalar_t>(bc, act, alpha, gain, clamp, bias_gain);
    OptTensor partial;
    int groups = 0;
    if (curved && !z) {
      // z again, from the product that made it
      const int64_t width = (n + 7) / 8 * 8;
      Rows dz{torch::empty({m, width}, x.options()), m, width};
      e.dy = cptr<scalar_t>(dr.t);
      e.dy_stride = dr.stride;
      groups = gfa::linear_row_tiles(m, n);
      if (need_db) partial = torch::empty({groups, n}, f32);
      e.partial = mptr<float>(partial);
      gfa::launch_linear_slope<scalar_t>(
          static_cast<scalar_t*>(dz.t.data_ptr()), cptr<scalar_t>(xr.t),
          cptr<scalar_t>(wr.t),
          {m, n, k, xr.stride, wr.stride, width, (float)weight_gain, k}, e,
          cur_stream());
      dr = dz;
    } else if (curved || need_db) {
      const int64_t width = (n + 7) / 8 * 8;
      Rows dz{Tensor(), m, width};
      if (curved) dz.t = torch::empty({m, width}, x.options());
      groups = gfa::linear_dz_groups(m, (int)n);
      if (need_db) partial = torch::empty({groups, n}, f32);
      gfa::launch_linear_dz<scalar_t>(
          curved ? static_cast<scalar_t*>(dz.t.data_ptr()) : nullptr, width,
          mptr<float>(partial), cptr<scalar_t>(dr.t), dr.stride,
          curved ? mptr<float>(z) : nullptr, e.act, m, (int)n, cur_stream());
      if (curved) dr = dz;
    }
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
    const float scale = (float)(weight_gain * slope);
    if (need_dx || need_dw) dr = tile_rows<scalar_t>(dr, n);
    if (need_dx)
      gfa::launch_linear_dx<scalar_t>(
          mptr<scalar_t>(dx), cptr<scalar_t>(dr.t), cptr<scalar_t>(wr.t),
          {m, k, n, dr.stride, wr.stride, k, scale, n}, cur_stream());
    if (need_dw) {
      const int splits =
          gfa::linear_splits(n, k, m, std::is_same_v<scalar_t, float>);
      OptTensor parts;
      if (splits > 1) parts = torch::empty({splits, n, k}, f32);
      gfa::launch_linear_dw<scalar_t>(
          mptr<scalar_t>(dw), mptr<float>(parts), cptr<scalar_t>(dr.t),
          cptr<scalar_t>(xr.t),
          {n, k, m, dr.stride, xr.stride, k, scale, m}, cur_stream());
    }
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
