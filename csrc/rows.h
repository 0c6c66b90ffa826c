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

// f(v[j]) for eight values behind one switch over the activation.
// Comparisons are written so that a NaN takes the branch that keeps it.
template <int N>
GFA_DEV void act_values(float (&z)[N], const ActParams& p) {
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = f(z[j]);
  };
  switch (p.act) {
    case kRelu: each([](float z) { return z <= 0.f ? 0.f : z; }); break;
    case kLrelu:
      each([&](float z) { return z <= 0.f ? p.alpha * z : z; });
      break;
    case kTanh: each([](float z) { return tanhf(z); }); break;
    case kSigmoid: each([](float z) { return 1.f / (1.f + expf(-z)); }); break;
    case kGelu:
      each([](float z) { return 0.5f * z * (1.f + erff(z * 0.70710678f)); });
      break;
    case kSilu: each([](float z) { return z / (1.f + expf(-z)); }); break;
  }
  each([&](float a) {
    a *= p.gain;
    return a > p.clamp ? p.clamp : a < -p.clamp ? -p.clamp : a;
  });
}

// d y / d z at z, zero where the clamp holds
template <int N>
GFA_DEV void act_slopes(float (&z)[N], const ActParams& p) {
  // f: activation and slope
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float a, s;
      f(z[j], a, s);
      z[j] = fabsf(a * p.gain) >= p.clamp ? 0.f : s * p.gain;
    }
  };
  switch (p.act) {
    case kLinear:
      each([](float z, float& a, float& s) { s = 1.f, a = z; });
      break;
    case kRelu:
      each([](float z, float& a, float& s) {
        s = z <= 0.f ? 0.f : 1.f, a = s * z;
      });
      break;
    case kLrelu:
      each([&](float z, float& a, float& s) {
        s = z <= 0.f ? p.alpha : 1.f, a = s * z;
      });
      break;
    case kTanh:
      each([](float z, float& a, float& s) {
        a = tanhf(z), s = 1.f - a * a;
      });
      break;
    case kSigmoid:
      each([](float z, float& a, float& s) {
        a = 1.f / (1.f + expf(-z)), s = a * (1.f - a);
      });
      break;
    case kGelu:
      each([](float z, float& a, float& s) {
        const float cdf = 0.5f * (1.f + erff(z * 0.70710678f));
        a = z * cdf, s = cdf + z * 0.39894228f * expf(-0.5f * z * z);
      });
      break;
    case kSilu:
      each([](float z, float& a, float& s) {
        const float g = 1.f / (1.f + expf(-z));
        a = z * g, s = g * (1.f + z * (1.f - g));
      });
      break;
  }
}

GFA_DEV float act_slope(float z, const ActParams& p) {
  float v[1] = {z};
  act_slopes(v, p);
  return v[0];
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

// C[m, n] = epilogue(alpha * sum_k A[m, k] B[n, k]). lda, ldb: strides of
// the operands' rows (or columns), multiples of 16 bytes below 2^20.
struct GemmArgs {
  long M, N, K;
  long lda, ldb, ldc;
  float alpha;
  long k_split;  // k of one split, a multiple of the tiles' depth
};
enum Epilogue { kPlain = 0, kForward, kSlope, kPartial };
template <typename T>
struct EpilogueArgs {
  const void* bias;  // [N] or null
  bool bias_f32;
  float bias_gain;
  ActParams act;
  const T* residual;  // forward: [M, N] with rows of res_stride, or null
  long res_stride;
  float* z;     // forward: [M, N] or null
  const T* dy;  // slope: [M, N] with rows of dy_stride
  long dy_stride;
  // slope: sums over the rows of each row of tiles, or null; with k in
  // parts: their sums
  float* partial;
};
// Into how many parts the launches below share k, given C's M x N: each but
// linear_slope takes linear_splits(...), and needs partial (e.partial) of
// that many M * N floats if it is over 1.
int linear_splits(long M, long N, long K, bool f32, bool dw);
// y = clamp(act(alpha x W^T + bias) * gain) + residual
template <typename T>
void launch_linear_forward(T* y, const T* x, const T* w, const GemmArgs& g,
                           const EpilogueArgs<T>& e, int splits, hipStream_t);
// dz = dy * slope(alpha x W^T + bias); linear_row_tiles sums of rows
int linear_row_tiles(long M, long N);
template <typename T>
void launch_linear_slope(T* dz, const T* x, const T* w, const GemmArgs& g,
                         const EpilogueArgs<T>& e, hipStream_t);
// dx[M, N] = alpha dz[M, K] W[K, N]
template <typename T>
void launch_linear_dx(T* dx, float* partial, const T* dz, const T* w,
                      const GemmArgs& g, int splits, hipStream_t);
// dw[M, N] = alpha dz[K, M]^T x[K, N]
template <typename T>
void launch_linear_dw(T* dw, float* partial, const T* dz, const T* x,
                      const GemmArgs& g, int splits, hipStream_t);
template <typename T>
void launch_pad_rows(T* dst, const T* src, long stride, long rows, int n,
                     int width, hipStream_t);

// dz = dy * slope(z) (z and dz null: dz = dy) and, unless partial is null,
// partial[g][n] = sums of dz over the rows of group g
int linear_dz_groups(long rows, int n);
template <typename T>
void launch_linear_dz(T* dz, long dz_stride, float* partial, const T* dy,
                      long dy_stride, const float* z, const ActParams& act,
                      long rows, int n, hipStream_t s);

}  // namespace gfa
