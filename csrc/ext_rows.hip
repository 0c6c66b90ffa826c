// Torch bindings of the row operators: layer_norm and linear_act.
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>

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

// Arguments that do not fit raise ValueError, as the Python side does.
#define CHECK_ARG TORCH_CHECK_VALUE

void check_device(const Tensor& t, const Tensor& x, const char* op,
                  const char* what) {
  CHECK_ARG(t.device() == x.device(), op, ": ", what, " is on ", t.device(),
            ", x on ", x.device());
}

void check_x(const Tensor& x, const char* op) {
  CHECK_ARG(x.is_cuda() && (x.scalar_type() == torch::kFloat32 ||
                            x.scalar_type() == torch::kBFloat16),
            op, ": expected float32 or bfloat16 on the GPU, got ",
            x.scalar_type(), " on ", x.device());
}

void check_param(const OptTensor& p, const Tensor& x, int64_t n,
                 const char* op, const char* what) {
  if (!p) return;
  CHECK_ARG(p->dim() == 1 && p->size(0) == n, op, ": ", what,
            ": expected shape [", n, "], got ", p->sizes());
  check_device(*p, x, op, what);
  CHECK_ARG(p->scalar_type() == x.scalar_type() ||
                p->scalar_type() == torch::kFloat32,
            op, ": ", what, ": expected ", x.scalar_type(),
            " or float32, got ", p->scalar_type());
}

// torch::empty without the way through the dispatcher, which costs more than
// the allocation
Tensor new_tensor(torch::IntArrayRef shape, torch::ScalarType dtype,
                  const Tensor& like) {
  return Tensor(at::detail::empty_cuda(shape, dtype, like.device(),
                                       std::nullopt));
}

// Room for a launch's intermediate values, on the current stream as tensors
// are: given back to the allocator at the end of its scope, reused only by
// what comes later on that stream.
struct Room {
  c10::DataPtr data;
  template <typename T>
  T* get(int64_t count) {
    if (count == 0) return nullptr;
    data = c10::hip::HIPCachingAllocator::get()->allocate(count * sizeof(T));
    return static_cast<T*>(data.get());
  }
};

// A tensor [..., n] as rows of n contiguous elements at one stride
struct Rows {
  Tensor t;  // what is read: the tensor itself or a contiguous copy
  int64_t count, stride;
  const void* at;
};

Rows rows_of(const Tensor& t) {
  const int64_t n = t.size(-1);
  Rows r{t, 1, n, t.data_ptr()};
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
    r.at = r.t.data_ptr();
  }
  return r;
}

template <typename T>
const T* rptr(const Rows& r) {
  return static_cast<const T*>(r.at);
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
  return w ? w->scalar_type() == torch::kFloat32
           : !b || b->scalar_type() == torch::kFloat32;
}

void check_layer_norm(const Tensor& x, const OptTensor& w,
                      const OptTensor& b) {
  const char* op = "layer_norm";
  check_x(x, op);
  CHECK_ARG(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1 << 30), op,
            ": x needs a last dimension of at least 1 (and below 2^30), got "
            "shape ", x.sizes());
  check_param(w, x, x.size(-1), op, "weight");
  check_param(b, x, x.size(-1), op, "bias");
  CHECK_ARG(!w || !b || w->scalar_type() == b->scalar_type(), op,
            ": weight is ", w->scalar_type(), ", bias ", b->scalar_type());
}

// y and, if they are to be kept, the means and the 1 / deviations [2, rows]
std::tuple<Tensor, OptTensor> layer_norm_fwd(
    const Tensor& x, const OptTensor& w, const OptTensor& b, double eps,
    bool save) {
  const int n = (int)x.size(-1);
  const bool p32 = params_f32(w, b);
  c10::hip::HIPGuard guard(x.get_device());
  const OptTensor wc = w ? OptTensor(w->contiguous()) : w;
  const OptTensor bc = b ? OptTensor(b->contiguous()) : b;
  const Rows xr = rows_of(x);
  Tensor y = new_tensor(x.sizes(), x.scalar_type(), x);
  OptTensor stats;
  if (save) {
    stats = new_tensor({2, xr.count}, torch::kFloat32, x);
  }
  if (xr.count > 0) {
    DISPATCH_TP(x, p32, {
      gfa::launch_layer_norm_fwd<T, P>(
          static_cast<T*>(y.data_ptr()), mptr<float>(stats),
          save ? mptr<float>(stats) + xr.count : nullptr,
          rptr<T>(xr), xr.stride, cptr<P>(wc), cptr<P>(bc), xr.count, n,
          (float)eps, cur_stream());
    });
    HIP_CHECK_LAST();
  }
  return {y, stats};
}

std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_bwd(
    const Tensor& dy, const Tensor& x, const OptTensor& w, const OptTensor& b,
    const Tensor& stats, bool need_dx, bool need_dw, bool need_db) {
  TORCH_CHECK(dy.device() == x.device() && dy.sizes() == x.sizes() &&
                  dy.scalar_type() == x.scalar_type(),
              "layer_norm: dy does not fit x");
  const int n = (int)x.size(-1);
  const bool p32 = params_f32(w, b);
  c10::hip::HIPGuard guard(x.get_device());
  const OptTensor wc = w ? OptTensor(w->contiguous()) : w;
  const Rows xr = rows_of(x), dr = rows_of(dy);
  const auto ptype = p32 ? torch::kFloat32 : x.scalar_type();
  OptTensor dx, dw, db;
  Room partial;
  if (need_dx) dx = new_tensor(x.sizes(), x.scalar_type(), x);
  if (need_dw) dw = new_tensor({n}, ptype, x);
  if (need_db) db = new_tensor({n}, ptype, x);
  if (xr.count == 0) {
    if (need_dw) dw->zero_();
    if (need_db) db->zero_();
    return {dx, dw, db};
  }
  const bool f32 = x.scalar_type() == torch::kFloat32;
  const bool by_sums = (need_dw || need_db) &&
                       gfa::layer_norm_bwd_sums(xr.count, n, f32);
  const int64_t groups = gfa::layer_norm_bwd_groups(xr.count, n, f32);
  float* sums = partial.get<float>(by_sums ? 2 * groups * n : 0);
  DISPATCH_TP(x, p32, {
    gfa::launch_layer_norm_bwd<T, P>(
        mptr<T>(dx), mptr<P>(dw), mptr<P>(db), sums,
        rptr<T>(dr), dr.stride, rptr<T>(xr), xr.stride, cptr<P>(wc),
        cptr<float>(stats), cptr<float>(stats) + xr.count, xr.count, n,
        cur_stream());
  });
  HIP_CHECK_LAST();
  return {dx, dw, db};
}

// ---- linear ----

void check_linear(const Tensor& x, const Tensor& w, const OptTensor& bias,
                  const OptTensor& residual) {
  const char* op = "linear_act";
  check_x(x, op);
  CHECK_ARG(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1), op,
            ": x ", x.sizes(), " and weight ", w.sizes(), " do not fit");
  CHECK_ARG(w.size(0) >= 1 && w.size(1) >= 1, op, ": empty weight ",
            w.sizes());
  CHECK_ARG(w.size(0) < (1 << 20) && w.size(1) < (1 << 20), op,
            ": weight of ", w.sizes(), ": sizes below 2^20 are served");
  CHECK_ARG(x.numel() / x.size(-1) < (1l << 30), op, ": x ", x.sizes(),
            ": fewer than 2^30 rows are served");
  check_device(w, x, op, "weight");
  CHECK_ARG(w.scalar_type() == x.scalar_type(), op, ": weight is ",
            w.scalar_type(), ", x ", x.scalar_type());
  check_param(bias, x, w.size(0), op, "bias");
  if (!residual) return;
  CHECK_ARG(residual->dim() == x.dim() && residual->size(-1) == w.size(0) &&
                residual->sizes().slice(0, x.dim() - 1) ==
                    x.sizes().slice(0, x.dim() - 1),
            op, ": residual ", residual->sizes(), " does not fit the output");
  check_device(*residual, x, op, "residual");
  CHECK_ARG(residual->scalar_type() == x.scalar_type(), op, ": residual is ",
            residual->scalar_type(), ", x ", x.scalar_type());
}

struct LinearParams {
  int64_t act;
  double alpha, gain, clamp, weight_gain, bias_gain;
  // Without an activation or a clamp the slope is the gain everywhere.
  bool curved() const { return act != gfa::kLinear || !std::isinf(clamp); }
};

std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
  auto s = x.sizes().vec();
  s.back() = n;
  return s;
}

// The tiles read rows of 16-byte granules: rows elsewhere, or of another
// width, are copied to padded ones (zeros behind the last element). So are rows
// that repeat or overlap where a product sums over them (`summed`): the last
// tile's end is found by the operand's, which has to lie before the row after
// the last. Up to two tensors in one launch.
template <typename T>
struct TileRows {
  Room room;
  gfa::PadArgs<T> pad{};

  void add(Rows& r, int64_t n, bool summed = false) {
    const int64_t v = 16 / sizeof(T);
    if (n % v == 0 && r.stride % v == 0 && r.stride < (1 << 20) &&
        (!summed || r.stride >= n) &&
        reinterpret_cast<uintptr_t>(r.at) % 16 == 0)
      return;
    const int64_t width = (n + 7) / 8 * 8;
    T* dst = room.get<T>(r.count * width);
    pad = {dst, static_cast<const T*>(r.at), r.stride, r.count, (int)n,
           (int)width};
    r.stride = width;
    r.at = dst;
  }
};

template <typename T>
void pad(const TileRows<T>& a, const TileRows<T>& b = {}) {
  if (a.pad.dst)
    gfa::launch_pad_rows<T>(a.pad, b.pad, cur_stream());
  else if (b.pad.dst)
    gfa::launch_pad_rows<T>(b.pad, a.pad, cur_stream());
}

template <typename T>
gfa::EpilogueArgs<T> epilogue(const OptTensor& bias, const LinearParams& p) {
  gfa::EpilogueArgs<T> e{};
  if (bias) {
    e.bias = bias->data_ptr();
    e.bias_f32 = bias->scalar_type() == torch::kFloat32;
    e.bias_gain = (float)p.bias_gain;
  }
  e.act = {(int)p.act, (float)p.alpha, (float)p.gain, (float)p.clamp};
  return e;
}

std::tuple<Tensor, OptTensor> linear_act_fwd(const Tensor& x, const Tensor& w,
                                             const OptTensor& bias,
                                             const OptTensor& residual,
                                             const LinearParams& p,
                                             bool save_z) {
  const int64_t n = w.size(0), k = w.size(1);
  const auto shape = out_shape(x, n);
  c10::hip::HIPGuard guard(x.get_device());
  const OptTensor bc = bias ? OptTensor(bias->contiguous()) : bias;
  Tensor y = new_tensor(shape, x.scalar_type(), x);
  OptTensor z;
  if (save_z) z = new_tensor(shape, torch::kFloat32, x);
  if (y.numel() == 0) return {y, z};
  DISPATCH_FT(x.scalar_type(), {
    Rows xr = rows_of(x), wr = rows_of(w);
    const int64_t m = xr.count;
    TileRows<scalar_t> px, pw;
    if (!gfa::linear_reads_any_rows(m)) {
      px.add(xr, k);
      pw.add(wr, k);
      pad(px, pw);
    }
    auto e = epilogue<scalar_t>(bc, p);
    Rows rr;
    if (residual) {
      rr = rows_of(*residual);
      e.residual = rptr<scalar_t>(rr);
      e.res_stride = rr.stride;
    }
    e.z = mptr<float>(z);
    const auto plan = gfa::linear_plan(
        m, n, k, std::is_same_v<scalar_t, float>, gfa::kRows);
    Room parts;
    e.partial = parts.get<float>(plan.splits > 1 ? plan.splits * m * n : 0);
    gfa::launch_linear_forward<scalar_t>(
        static_cast<scalar_t*>(y.data_ptr()), rptr<scalar_t>(xr),
        rptr<scalar_t>(wr),
        {m, n, k, xr.stride, wr.stride, n, (float)p.weight_gain, k}, e, plan,
        cur_stream());
  });
  HIP_CHECK_LAST();
  return {y, z};
}

std::tuple<OptTensor, OptTensor, OptTensor> linear_act_bwd(
    const Tensor& dy, const OptTensor& z, const Tensor& x, const Tensor& w,
    const OptTensor& bias, const LinearParams& p, bool need_dx, bool need_dw,
    bool need_db) {
  const int64_t n = w.size(0), k = w.size(1);
  TORCH_CHECK(dy.device() == x.device() && dy.sizes() == out_shape(x, n) &&
                  dy.scalar_type() == x.scalar_type(),
              "linear_act: dy does not fit");
  c10::hip::HIPGuard guard(x.get_device());
  const int64_t m = dy.numel() / n;
  OptTensor dx, dw, db;
  if (need_dx) dx = new_tensor(x.sizes(), x.scalar_type(), x);
  if (m == 0) {
    if (need_dw) dw = torch::zeros(w.sizes(), w.options());
    if (need_db) db = torch::zeros({n}, bias->options());
    return {dx, dw, db};
  }
  if (need_dw) dw = new_tensor(w.sizes(), w.scalar_type(), x);
  if (need_db) db = new_tensor({n}, bias->scalar_type(), x);
  if (!need_dx && !need_dw && !need_db) return {dx, dw, db};
  const OptTensor bc = bias ? OptTensor(bias->contiguous()) : bias;
  // a slope that is the same everywhere goes into the products: dz is dy
  const bool curved = p.curved(), again = curved && !z;
  const double slope = curved ? 1.0 : p.gain;
  const bool small = gfa::linear_backward_is_small(
      m, n, k, x.scalar_type() == torch::kFloat32);
  DISPATCH_FT(x.scalar_type(), {
    constexpr bool is_f32 = std::is_same_v<scalar_t, float>;
    Rows xr = rows_of(x), wr = rows_of(w), dr = rows_of(dy);
    TileRows<scalar_t> px, pw, pd;
    const bool any = gfa::linear_reads_any_rows(m);
    if (need_dw || (again && !any)) px.add(xr, k, need_dw);
    if (need_dx || (again && !any)) pw.add(wr, k, need_dx);
    pad(px, pw);
    auto e = epilogue<scalar_t>(bc, p);
    Room dz_room, partial_room, dx_parts, dw_parts;
    float* partial = nullptr;
    int groups = 0;
    if (curved) {
      const int64_t width = (n + 7) / 8 * 8;  // zeros behind n
      // a bf16 dz in two parts
      scalar_t* dz = dz_room.get<scalar_t>(m * width * (is_f32 ? 1 : 2));
      if (!is_f32) e.dz_low = dz + m * width;
      const auto plan = gfa::linear_plan(m, n, k, is_f32, gfa::kSlopes);
      groups = again ? gfa::linear_row_tiles(plan, m)
                     : gfa::linear_dz_groups(m, (int)n);
      partial = partial_room.get<float>(need_db ? groups * n : 0);
      if (again) {
        // z again, from the product that made it
        e.dy = rptr<scalar_t>(dr);
        e.dy_stride = dr.stride;
        e.partial = partial;
        gfa::launch_linear_slope<scalar_t>(
            dz, rptr<scalar_t>(xr), rptr<scalar_t>(wr),
            {m, n, k, xr.stride, wr.stride, width, (float)p.weight_gain, k}, e,
            plan, cur_stream());
      } else {
        gfa::launch_linear_dz<scalar_t>(dz, e.dz_low, width, partial,
                                        rptr<scalar_t>(dr), dr.stride,
                                        mptr<float>(z), e.act, m, (int)n,
                                        cur_stream());
      }
      dr.at = dz;
      dr.stride = width;
    } else {
      if (need_db && !small) {
        groups = gfa::linear_dz_groups(m, (int)n);
        partial = partial_room.get<float>(groups * n);
        gfa::launch_linear_dz<scalar_t>(nullptr, nullptr, 0, partial,
                                        rptr<scalar_t>(dr), dr.stride, nullptr,
                                        e.act, m, (int)n, cur_stream());
      }
      if (need_dx || need_dw) {
        pd.add(dr, n, need_dw);
        pad(pd);
      }
    }
    const float scale = (float)(p.weight_gain * slope);
    const float db_scale = (float)(p.bias_gain * slope);
    const bool db_f32 = need_db && bias->scalar_type() == torch::kFloat32;
    const gfa::GemmArgs gx{m, k, n, dr.stride, wr.stride, k, scale, n};
    const gfa::GemmArgs gw{n, k, m, dr.stride, xr.stride, k, scale, m};
    const int passes = e.dz_low ? 2 : 1;
    if (small) {
      gfa::SmallBackward<scalar_t> s{};
      s.dw = gw;
      s.dx = gx;
      s.dw_out = mptr<scalar_t>(dw);
      s.dx_out = mptr<scalar_t>(dx);
      s.db_out = db ? db->data_ptr() : nullptr;
      s.db_f32 = db_f32;
      s.dz = rptr<scalar_t>(dr);
      s.dz_low = e.dz_low;
      s.x = rptr<scalar_t>(xr);
      s.w = rptr<scalar_t>(wr);
      s.partial = partial;
      s.groups = groups;
      s.n = (int)n;
      s.db_scale = db_scale;
      gfa::launch_linear_backward_small<scalar_t>(s, cur_stream());
    } else {
      if (db_f32)
        gfa::launch_sum_groups<float>(mptr<float>(db), nullptr, partial,
                                      groups, (int)n, db_scale, cur_stream());
      else if (need_db)
        gfa::launch_sum_groups<gfa::bf16>(mptr<gfa::bf16>(db), nullptr,
                                          partial, groups, (int)n, db_scale,
                                          cur_stream());
      if (need_dx) {
        const auto plan =
            gfa::linear_plan(m, k, n * passes, is_f32, gfa::kInputs);
        gfa::launch_linear_dx<scalar_t>(
            mptr<scalar_t>(dx),
            dx_parts.get<float>(plan.splits > 1 ? plan.splits * m * k : 0),
            rptr<scalar_t>(dr), e.dz_low, rptr<scalar_t>(wr), gx, plan,
            cur_stream());
      }
      if (need_dw) {
        const auto plan =
            gfa::linear_plan(n, k, m * passes, is_f32, gfa::kWeights);
        gfa::launch_linear_dw<scalar_t>(
            mptr<scalar_t>(dw),
            dw_parts.get<float>(plan.splits > 1 ? plan.splits * n * k : 0),
            rptr<scalar_t>(dr), e.dz_low, rptr<scalar_t>(xr), gw, plan,
            cur_stream());
      }
    }
  });
  HIP_CHECK_LAST();
  return {dx, dw, db};
}

// ---- autograd ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptTensor opt(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}
Tensor plain(const OptTensor& t) { return t ? *t : Tensor(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }

// Which of the tensors (null: not given) need a gradient. The context counts
// only those that are there.
std::vector<bool> needed(AutogradContext* ctx, const variable_list& in) {
  std::vector<bool> need;
  size_t k = 0;
  for (const Tensor& t : in)
    need.push_back(t.defined() && ctx->needs_input_grad(k++));
  return need;
}

// Whether a backward is itself differentiated, in reverse or forward mode
bool differentiated(const Tensor& dy) {
  return torch::GradMode::is_enabled() || torch::autograd::isFwGradDefined(dy);
}

// Differentiable gradients of f(inputs) in those that need one, for such a
// backward: of the inputs without the residual, whose gradient is dy. Through
// a view of each input: one may come from another (a residual and what was
// made from it), and this operator's gradient must not run on into that
// history.
template <typename F>
variable_list composed_grads(const variable_list& in,
                             const std::vector<bool>& need, const Tensor& dy,
                             F&& f) {
  const bool again = torch::GradMode::is_enabled();
  torch::AutoGradMode graph(true);
  variable_list views, wanted;
  for (size_t i = 0; i < in.size(); ++i) {
    views.push_back(in[i].defined() ? in[i].view_as(in[i]) : Tensor());
    if (need[i]) wanted.push_back(views.back());
  }
  variable_list out(in.size());
  if (wanted.empty()) return out;
  const variable_list got = torch::autograd::grad(
      {f(views)}, wanted, {dy}, /*retain_graph=*/std::nullopt,
      /*create_graph=*/again);
  size_t k = 0;
  for (size_t i = 0; i < in.size(); ++i)
    if (need[i]) out[i] = got[k++];
  return out;
}

// Whether a call has to consist of torch's own operations: one of its tensors
// carries a forward-mode tangent, which the kernels would drop, or the call is
// traced, and a trace would hold their results as constants.
bool takes_composition(const Tensor& x, const OptTensor& a, const OptTensor& b,
                       const OptTensor& c = {}) {
  using torch::autograd::isFwGradDefined;
  return torch::jit::tracer::isTracing() || isFwGradDefined(x) ||
         isFwGradDefined(a) || isFwGradDefined(b) || isFwGradDefined(c);
}

Tensor composed_layer_norm(const variable_list& in, double eps) {
  const Tensor x = in[0].to(torch::kFloat32);
  const Tensor xc = x - x.mean(-1, true);
  Tensor y = xc * (xc.square().mean(-1, true) + eps).rsqrt();
  if (in[1].defined()) y = y * in[1];
  if (in[2].defined()) y = y + in[2];
  return y.to(in[0].scalar_type());
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x,
                        const OptTensor& w, const OptTensor& b, double eps) {
    auto [y, stats] = layer_norm_fwd(x, w, b, eps, true);
    ctx->save_for_backward({x, plain(w), plain(b), *stats});
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto s = ctx->get_saved_variables();
    const variable_list in{s[0], s[1], s[2]};
    const auto need = needed(ctx, in);
    if (differentiated(dy[0])) {
      const double eps = ctx->saved_data["eps"].toDouble();
      auto out = composed_grads(in, need, dy[0], [&](const variable_list& v) {
        return composed_layer_norm(v, eps);
      });
      out.emplace_back();
      return out;
    }
    const auto [dx, dw, db] =
        layer_norm_bwd(dy[0], s[0], opt(s[1]), opt(s[2]), s[3], need[0],
                       need[1], need[2]);
    return {plain(dx), plain(dw), plain(db), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& w, const OptTensor& b,
                  double eps) {
  check_layer_norm(x, w, b);
  if (takes_composition(x, w, b))
    return composed_layer_norm({x, plain(w), plain(b)}, eps);
  if (torch::GradMode::is_enabled() &&
      (x.requires_grad() || wants_grad(w) || wants_grad(b)))
    return LayerNorm::apply(x, w, b, eps);
  return std::get<0>(layer_norm_fwd(x, w, b, eps, false));
}

Tensor composed_linear_act(const variable_list& in, const LinearParams& p,
                           const OptTensor& residual = {}) {
  Tensor z = torch::matmul(in[0].to(torch::kFloat32),
                           in[1].to(torch::kFloat32).t()) * p.weight_gain;
  if (in[2].defined()) z = z + in[2].to(torch::kFloat32) * p.bias_gain;
  Tensor y = z;
  switch (p.act) {
    case gfa::kRelu: y = torch::relu(z); break;
    case gfa::kLrelu: y = torch::leaky_relu(z, p.alpha); break;
    case gfa::kTanh: y = torch::tanh(z); break;
    case gfa::kSigmoid: y = torch::sigmoid(z); break;
    case gfa::kGelu: y = z * 0.5 * (1.0 + torch::erf(z * M_SQRT1_2)); break;
    case gfa::kSilu: y = z * torch::sigmoid(z); break;
  }
  y = y * p.gain;
  // clamp's own gradient would pass where y just reaches it; the kernels' and
  // bias_act's is 0 there
  if (!std::isinf(p.clamp))
    y = torch::where(y.abs() >= p.clamp, y.detach().clamp(-p.clamp, p.clamp),
                     y);
  if (residual) y = y + *residual;
  return y.to(in[0].scalar_type());
}

// Whether the forward keeps z for the backward, in 32 bits (a rounded z
// would cost the slopes, and the bias's gradient, their digits). Keeping it
// moves 8 bytes an element and a pass over dz; computing it again costs k
// multiplications an element and happens where dz is made. The two meet at
// about 1500 (bf16) and 128 (float) multiplications.
bool keeps_z(const Tensor& x, const Tensor& w, const OptTensor& bias,
             const LinearParams& p) {
  return p.curved() &&
         (x.requires_grad() || w.requires_grad() || wants_grad(bias)) &&
         x.size(-1) > (x.scalar_type() == torch::kFloat32 ? 128 : 1536);
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const OptTensor& bias, const OptTensor& residual,
                        const LinearParams& p) {
    auto [y, z] =
        linear_act_fwd(x, w, bias, residual, p, keeps_z(x, w, bias, p));
    // the residual, whose gradient is dy, is not needed again
    ctx->save_for_backward({x, w, plain(bias), plain(z)});
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["params"] =
        std::vector<double>{(double)p.act, p.alpha,       p.gain,
                            p.clamp,       p.weight_gain, p.bias_gain};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto s = ctx->get_saved_variables();
    const auto d = ctx->saved_data["params"].toDoubleVector();
    const LinearParams p{(int64_t)d[0], d[1], d[2], d[3], d[4], d[5]};
    const variable_list in{s[0], s[1], s[2]};
    const auto need = needed(ctx, in);
    const Tensor dres = ctx->saved_data["residual"].toBool() &&
                                ctx->needs_input_grad(s[2].defined() ? 3 : 2)
                            ? dy[0]
                            : Tensor();
    if (differentiated(dy[0])) {
      auto out = composed_grads(in, need, dy[0], [&](const variable_list& v) {
        return composed_linear_act(v, p);
      });
      out.push_back(dres);
      out.emplace_back();
      return out;
    }
    const auto [dx, dw, db] =
        linear_act_bwd(dy[0], opt(s[3]), s[0], s[1], opt(s[2]), p, need[0],
                       need[1], need[2]);
    return {plain(dx), plain(dw), plain(db), dres, Tensor()};
  }
};

Tensor linear_act(const Tensor& x, const Tensor& w, const OptTensor& bias,
                  const OptTensor& residual, int64_t act, double alpha,
                  double gain, double clamp, double weight_gain,
                  double bias_gain) {
  check_linear(x, w, bias, residual);
  CHECK_ARG(act >= 0 && act <= gfa::kSilu, "linear_act: activation ", act);
  const LinearParams p{act, alpha, gain, clamp, weight_gain, bias_gain};
  if (takes_composition(x, w, bias, residual))
    return composed_linear_act({x, w, plain(bias)}, p, residual);
  if (torch::GradMode::is_enabled() &&
      (x.requires_grad() || w.requires_grad() || wants_grad(bias) ||
       wants_grad(residual)))
    return LinearAct::apply(x, w, bias, residual, p);
  return std::get<0>(linear_act_fwd(x, w, bias, residual, p, false));
}

}  // namespace

void bind_rows(pybind11::module& m) {
  m.def("layer_norm", &layer_norm, "layer norm over the last dimension");
  m.def("linear_act", &linear_act,
        "clamp(act(wg x W^T + bg b) * gain) + residual");
}
