// Shared by the row operators (layer_norm.hip, linear_act.hip) and their
// bindings (ext_rows.hip).
#pragma once

#include "common.h"

namespace gfa {

// rounding to T in hardware, to nearest even, NaN kept
template <typename T> GFA_DEV typename Raw<T>::type round_raw(float v);
template <> GFA_DEV float round_raw<float>(float v) { return v; }
template <> GFA_DEV u16 round_raw<bf16>(float v) {
  return __builtin_bit_cast(u16, static_cast<__bf16>(v));
}
template <typename T> GFA_DEV void put(T* p, float v) {
  *reinterpret_cast<typename Raw<T>::type*>(p) = round_raw<T>(v);
}

// activation codes of gansformer_amd/ops/linear_act.py
enum Act { kLinear = 0, kRelu, kLrelu, kTanh, kSigmoid, kGelu, kSilu };

struct ActParams {
  int act;
  float alpha, gain, clamp;  // clamp: infinity for none
};

// Comparisons are written so that a NaN takes the branch that keeps it.
GFA_DEV float act_value(float z, const ActParams& p) {
  float a = z;
  switch (p.act) {
    case kRelu: a = z <= 0.f ? 0.f : z; break;
    case kLrelu: a = z <= 0.f ? p.alpha * z : z; break;
    case kTanh: a = tanhf(z); break;
    case kSigmoid: a = 1.f / (1.f + expf(-z)); break;
    case kGelu: a = 0.5f * z * (1.f + erff(z * 0.70710678f)); break;
    case kSilu: a = z / (1.f + expf(-z)); break;
  }
  a *= p.gain;
  return a > p.clamp ? p.clamp : a < -p.clamp ? -p.clamp : a;
}

// d y / d z at z, zero where the clamp holds
GFA_DEV float act_slope(float z, const ActParams& p) {
  float a = z, s = 1.f;
  switch (p.act) {
    case kRelu:
      s = z <= 0.f ? 0.f : 1.f;
      a = s * z;
      break;
    case kLrelu:
      s = z <= 0.f ? p.alpha : 1.f;
      a = s * z;
      break;
    case kTanh:
      a = tanhf(z);
      s = 1.f - a * a;
      break;
    case kSigmoid:
      a = 1.f / (1.f + expf(-z));
      s = a * (1.f - a);
      break;
    case kGelu: {
      const float cdf = 0.5f * (1.f + erff(z * 0.70710678f));
      a = z * cdf;
      s = cdf + z * 0.39894228f * expf(-0.5f * z * z);
      break;
    }
    case kSilu: {
      const float g = 1.f / (1.f + expf(-z));
      a = z * g;
      s = g * (1.f + z * (1.f - g));
      break;
    }
  }
  return fabsf(a * p.gain) >= p.clamp ? 0.f : s * p.gain;
}

// T: float or bf16. P: type of the parameters (null pointer for none).
template <typename T, typename P>
void launch_layer_norm_fwd(T* y, float* mean, float* rstd, const T* x,
                           long x_stride, const P* w, const P* b, long rows,
                           int n, float eps, hipStream_t);
// partial: [2][groups][n] floats; dx, dw, db null if not wanted
int layer_norm_bwd_groups(long rows, int n, bool f32);
template <typename T, typename P>
void launch_layer_norm_bwd(T* dx, P* dw, P* db, float* partial, const T* dy,
                           long dy_stride, const T* x, long x_stride,
                           const P* w, const float* mean, const float* rstd,
                           long rows, int n, hipStream_t);

// out_k[i] = scale * sum_g partial[k][g][i], k = 0, 1; an out may be null
template <typename P>
void launch_sum_groups(P* out0, P* out1, const float* partial, int groups,
                       int n, float scale, hipStream_t);

// C[m, n] = epilogue(alpha * sum_k A[m, k] B[n, k]); one of the two strides
// of A and of B is 1
struct GemmArgs {
  long M, N, K;
  long sam, sak;  // strides of A
  long sbn, sbk;  // strides of B
  float alpha;
};
template <typename T>
struct EpilogueArgs {
  const void* bias;  // [N] or null
  bool bias_f32;
  float bias_gain;
  const T* residual;  // [M, N] with rows of res_stride, or null
  long res_stride;
  T* z;  // [M, N] or null
  ActParams act;
};
template <typename T>
void launch_linear_gemm(T* c, const T* a, const T* b, const GemmArgs& g,
                        const EpilogueArgs<T>& e, hipStream_t);

// dz = dy * slope(z) (z and dz null: dz = dy) and, unless partial is null,
// partial[g][n] = sums of dz over the rows of group g
int linear_dz_groups(long rows, int n);
template <typename T>
void launch_linear_dz(T* dz, float* partial, const T* dy, long dy_stride,
                      const T* z, const ActParams& act, long rows, int n,
                      hipStream_t);

}  // namespace gfa
