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

// v in two bf16 numbers whose sum is v up to 2^-15 of it: what is left of it
// toward zero, and the rest. Both have v's sign and, unless v is 0, neither is
// 0: a product with an infinity stays that infinity, where rests of the other
// sign or 0 would make the sum of both products no number. So does an infinite
// v, which has no rest. (A NaN that a product made has its first bit below
// the exponent set: it stays one.)
GFA_DEV void split(float v, u16& high, float& rest) {
  constexpr float kLeast = 1.17549435e-38f;  // smallest normal number
  high = (u16)(__float_as_uint(v) >> 16);
  rest = v - raw_to_f32(high);
  if (!(fabsf(rest) >= kLeast && fabsf(rest) < INFINITY))
    rest = v == 0.f ? 0.f : copysignf(kLeast, v);
}

// activation codes of gansformer_amd/ops/linear_act.py
enum Act { kLinear = 0, kRelu, kLrelu, kTanh, kSigmoid, kGelu, kSilu };

struct ActParams {
  int act;
  float alpha, gain, clamp;  // clamp: infinity for none
};

// ---- activations ----
// On the hardware's exponential and reciprocal (one unit in the last place
// each): the library's erf and tanh are several times as many instructions,
// and a product of few multiplications an element is bounded by them.
// An exponential's argument is rounded besides, so its relative error grows
// with the argument. Measured against 64 bits over |z| <= 12, relative for the
// values and absolute for the slopes, in units of 1e-7:
//            |z| <= 2     2..4        4..8        8..12
//   gelu     5.5, 2.4     8.7, 1.1    28, 0.9     75 (below 1e-14), 0
//   silu     2.5, 1.5     3.6, 3.6    5.5, 7.1    9.4, 7.7
//   tanh     1.8, 1.3     0.4, 0.3    0.3, 0      0.3, 0
//   sigmoid  2.2, 0.8     3.2, 1.1    5.4, 1.0    9.1, 0.9
GFA_DEV float fast_exp(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
GFA_DEV float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + fast_exp(-z));
}

// The normal distribution's upper tail at |z|, and exp(-z^2 / 2): the tail is
// exp(-u^2 / 2) P(1 / (1 + 0.304 u)) with a polynomial P fitted to it for u
// in 0..14 (largest relative error of the fit alone 9.6e-8).
GFA_DEV float normal_tail(float z, float& bell) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.304f * fabsf(z));
  bell = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  float p = 0.036624051934627824f;
  p = p * t - 0.15434850690885712f;
  p = p * t + 0.19059470868362968f;
  p = p * t - 0.04170049739369904f;
  p = p * t + 0.12281604221320018f;
  p = p * t + 0.10264079618297697f;
  p = p * t + 0.1221365383297614f;
  p = p * t + 0.12123686701196146f;
  return p * (t * bell);
}

// tanh(z), and 1 - tanh(z)^2 = 4 r (1 - r) with r = 1 / (1 + exp(2 |z|)).
// Below 0.6 by a polynomial in z^2 (relative error of the fit alone 2.5e-9),
// where 1 - 2 r would lose digits.
GFA_DEV float tanh_of(float z, float& slope) {
  const float r = __builtin_amdgcn_rcpf(1.f + fast_exp(2.f * fabsf(z)));
  slope = 4.f * r * (1.f - r);
  const float s = z * z;
  float p = -0.005852152574643519f;
  p = p * s + 0.020753615804063843f;
  p = p * s - 0.053768701016077794f;
  p = p * s + 0.13331688918204498f;
  p = p * s - 0.3333328325571884f;
  p = p * s + 0.9999999975108838f;
  return s < 0.36f ? z * p : copysignf(1.f - 2.f * r, z);
}

// f(v[j]) for all values behind one switch over the activation.
// Comparisons are written so that a NaN takes the branch that keeps it.
template <int N>
GFA_DEV void act_values(float (&z)[N], const ActParams& p) {
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = f(z[j]);
  };
  float unused;
  switch (p.act) {
    case kRelu: each([](float z) { return z <= 0.f ? 0.f : z; }); break;
    case kLrelu:
      each([&](float z) { return z <= 0.f ? p.alpha * z : z; });
      break;
    case kTanh: each([&](float z) { return tanh_of(z, unused); }); break;
    case kSigmoid: each([](float z) { return sigmoid(z); }); break;
    case kGelu:
      // z Phi(z), without a difference of nearly equal numbers on either side;
      // past 16 the tail is 0, and z, which may be infinite, does not meet it.
      // fmaxf and fminf drop a NaN, the tail keeps it.
      each([&](float z) {
        const float q = normal_tail(z, unused);
        return fmaxf(z, 0.f) - fabsf(fminf(z, 16.f)) * q;
      });
      break;
    case kSilu: each([](float z) { return z * sigmoid(z); }); break;
  }
  if (p.gain != 1.f) each([&](float a) { return a * p.gain; });
  if (p.clamp < INFINITY)
    each([&](float a) {
      return a > p.clamp ? p.clamp : a < -p.clamp ? -p.clamp : a;
    });
}

// d y / d z at z, zero where the clamp holds
template <int N>
GFA_DEV void act_slopes(float (&z)[N], const ActParams& p) {
  // f: activation and slope
  auto each = [&](auto f) {
    if (p.clamp < INFINITY) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float a, s;
        f(z[j], a, s);
        z[j] = fabsf(a * p.gain) >= p.clamp ? 0.f : s * p.gain;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float a, s;
        f(z[j], a, s);
        z[j] = s * p.gain;
      }
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
      each([](float z, float& a, float& s) { a = tanh_of(z, s); });
      break;
    case kSigmoid:
      each([](float z, float& a, float& s) {
        a = sigmoid(z), s = a * (1.f - a);
      });
      break;
    case kGelu:
      each([](float z, float& a, float& s) {
        float bell;
        const float q = normal_tail(z, bell);
        const float cdf = z < 0.f ? q : 1.f - q;
        a = z * cdf, s = cdf + z * 0.39894228f * bell;
      });
      break;
    case kSilu:
      each([](float z, float& a, float& s) {
        const float g = sigmoid(z);
        a = z * g, s = g * (1.f + z * (1.f - g));
      });
      break;
  }
}

// T: float or bf16. P: type of the parameters (null pointer for none).
template <typename T, typename P>
void launch_layer_norm_fwd(T* y, float* mean, float* rstd, const T* x,
                           long x_stride, const P* w, const P* b, long rows,
                           int n, float eps, hipStream_t);
// dx, dw, db null if not wanted. partial: [2][groups][n] floats, where dw and
// db go by sums of blocks and one is wanted; else null.
bool layer_norm_bwd_sums(long rows, int n, bool f32);
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
// the operands' rows (or columns), multiples of 16 bytes below 2^20; of
// columns, no shorter than M or N.
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
  T* dz_low;    // slope: the rest of a bf16 dz (split)
  const T* a_low;  // dx, dw: that rest, the left operand a second time, or null
  const T* dy;  // slope: [M, N] with rows of dy_stride
  long dy_stride;
  // slope: sums over the rows of each row of tiles, or null; with k in
  // parts: their sums
  float* partial;
};
// How C's M x N are cut up for the launches below: the side of a tile, and
// into how many parts k is shared. For more than one, partial (e.partial)
// holds that many M * N floats.
struct LinearPlan {
  int tile, splits;
};
enum LinearKind { kRows, kSlopes, kInputs, kWeights };
LinearPlan linear_plan(long M, long N, long K, bool f32, LinearKind kind);
// whether forward and slope of M rows read x and W at any alignment
bool linear_reads_any_rows(long M);
// y = clamp(act(alpha x W^T + bias) * gain) + residual
template <typename T>
void launch_linear_forward(T* y, const T* x, const T* w, const GemmArgs& g,
                           const EpilogueArgs<T>& e, const LinearPlan&,
                           hipStream_t);
// dz = dy * slope(alpha x W^T + bias); linear_row_tiles sums of rows
int linear_row_tiles(const LinearPlan&, long M);
template <typename T>
void launch_linear_slope(T* dz, const T* x, const T* w, const GemmArgs& g,
                         const EpilogueArgs<T>& e, const LinearPlan&,
                         hipStream_t);
// dx[M, N] = alpha dz[M, K] W[K, N]; dz_low: the rest of dz, or null. The plan
// is that of a K twice as long where there is a rest.
template <typename T>
void launch_linear_dx(T* dx, float* partial, const T* dz, const T* dz_low,
                      const T* w, const GemmArgs& g, const LinearPlan&,
                      hipStream_t);
// dw[M, N] = alpha dz[K, M]^T x[K, N], likewise
template <typename T>
void launch_linear_dw(T* dw, float* partial, const T* dz, const T* dz_low,
                      const T* x, const GemmArgs& g, const LinearPlan&,
                      hipStream_t);
// dw, dx and db (each null if not wanted) of a small layer in one launch
template <typename T>
struct SmallBackward {
  GemmArgs dw, dx;
  T *dw_out, *dx_out;
  void* db_out;
  bool db_f32;
  const T *dz, *dz_low;  // dz_low: the rest of dz, or null
  const T *x, *w;
  // db: db_scale times the sums of the groups of partial, or of dz's rows
  const float* partial;
  int groups, n;
  float db_scale;
  int dw_blocks, dx_blocks;
};
bool linear_backward_is_small(long m, long n, long k, bool f32);
template <typename T>
void launch_linear_backward_small(SmallBackward<T> p, hipStream_t);

// dst [rows][width] = src [rows][n] at a stride, zero behind n; dst may be
// null. width is a multiple of 8.
template <typename T>
struct PadArgs {
  T* dst;
  const T* src;
  long stride, rows;
  int n, width;
};
template <typename T>
void launch_pad_rows(const PadArgs<T>& p0, const PadArgs<T>& p1, hipStream_t);

// dz = dy * slope(z) (z and dz null: dz = dy), low the rest of it if it is
// bf16 (split), and, unless partial is null,
// partial[g][n] = sums of dz over the rows of group g
int linear_dz_groups(long rows, int n);
template <typename T>
void launch_linear_dz(T* dz, T* low, long dz_stride, float* partial,
                      const T* dy,
                      long dy_stride, const float* z, const ActParams& act,
                      long rows, int n, hipStream_t s);

}  // namespace gfa
