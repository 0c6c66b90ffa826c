// Matrix product with bias, activation and residual in its epilogue, and
// the three products of its backward, for gfx950.
//
//   z  = alpha * A B^T + bias_gain * bias
//   y  = clamp(act(z) * gain) + residual
//   dz = dy * slope(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz
//
// Every product is one C[m, n] = sum_k A[m, k] B[n, k] over operands whose
// rows or whose columns are contiguous. Sums in float on the matrix cores;
// z, y and the gradients are rounded to T once, on their way out.
#include "rows.h"

namespace gfa {

// 64x64 tile, 4 waves of 32x32; any strides, any sizes.
template <typename T>
__global__ __launch_bounds__(256)
void linear_gemm_kernel(T* __restrict__ c, const T* __restrict__ a,
                        const T* __restrict__ b, GemmArgs g,
                        EpilogueArgs<T> e) {
  using TO = TileOps<T>;
  constexpr int BK = TO::BK;
  using elem = typename TO::elem;
  __shared__ elem As[64 * TO::ROW];
  __shared__ elem Bs[64 * TO::ROW];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const long m0 = (long)blockIdx.x * 64, n0 = (long)blockIdx.y * 64;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;

  f32x4 acc[2][2] = {};
  for (long k0 = 0; k0 < g.K; k0 += BK) {
    __syncthreads();
    for (int i = t; i < 64 * BK; i += 256) {
      // neighbouring threads along the contiguous dimension
      const int ra = g.sak == 1 ? i / BK : i % 64;
      const int ka = g.sak == 1 ? i % BK : i / 64;
      const bool oka = m0 + ra < g.M && k0 + ka < g.K;
      TO::store(As, ra, ka,
                oka ? to_f32(a[(m0 + ra) * g.sam + (k0 + ka) * g.sak]) : 0.f);
      const int rb = g.sbk == 1 ? i / BK : i % 64;
      const int kb = g.sbk == 1 ? i % BK : i / 64;
      const bool okb = n0 + rb < g.N && k0 + kb < g.K;
      TO::store(Bs, rb, kb,
                okb ? to_f32(b[(n0 + rb) * g.sbn + (k0 + kb) * g.sbk]) : 0.f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = TO::mfma(As, Bs, wm + i * 16, wn + j * 16, lane,
                             acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const long m = m0 + wm + i * 16 + (lane >> 4) * 4 + q;
        const long n = n0 + wn + j * 16 + (lane & 15);
        if (m >= g.M || n >= g.N) continue;
        float z = g.alpha * acc[i][j][q];
        if (e.bias)
          z += e.bias_gain * (e.bias_f32
                                  ? static_cast<const float*>(e.bias)[n]
                                  : to_f32(static_cast<const T*>(e.bias)[n]));
        if (e.z) put(e.z + m * g.N + n, z);
        float y = act_value(z, e.act);
        if (e.residual) y += to_f32(e.residual[m * e.res_stride + n]);
        put(c + m * g.N + n, y);
      }
}

template <typename T>
void launch_linear_gemm(T* c, const T* a, const T* b, const GemmArgs& g,
                        const EpilogueArgs<T>& e, hipStream_t s) {
  hipLaunchKernelGGL(linear_gemm_kernel<T>,
                     dim3(ceil_div(g.M, 64), ceil_div(g.N, 64)), dim3(256), 0,
                     s, c, a, b, g, e);
}

// thread: one column; block: 256 columns of one group of rows
template <typename T>
__global__ __launch_bounds__(256)
void linear_dz_kernel(T* __restrict__ dz, float* __restrict__ partial,
                      const T* __restrict__ dy, long dy_stride,
                      const T* __restrict__ z, ActParams act, long rows,
                      int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int groups = gridDim.y;
  const long per = (rows + groups - 1) / groups;
  const long r0 = blockIdx.y * per, r1 = min(r0 + per, rows);
  if (i >= n) return;
  float sum = 0.f;
  for (long r = r0; r < r1; ++r) {
    float d = to_f32(dy[r * dy_stride + i]);
    if (z) {
      d *= act_slope(to_f32(z[r * n + i]), act);
      put(dz + r * n + i, d);
    }
    sum += d;  // before its rounding
  }
  if (partial) partial[(long)blockIdx.y * n + i] = sum;
}

int linear_dz_groups(long rows, int n) {
  const long g = (rows + 63) / 64;
  return (int)(g < 256 ? g : 256);
}

template <typename T>
void launch_linear_dz(T* dz, float* partial, const T* dy, long dy_stride,
                      const T* z, const ActParams& act, long rows, int n,
                      hipStream_t s) {
  hipLaunchKernelGGL(linear_dz_kernel<T>,
                     dim3(ceil_div(n, 256), linear_dz_groups(rows, n)),
                     dim3(256), 0, s, dz, partial, dy, dy_stride, z, act,
                     rows, n);
}

#define INSTANTIATE(T)                                                       \
  template void launch_linear_gemm<T>(T*, const T*, const T*,                \
                                      const GemmArgs&,                       \
                                      const EpilogueArgs<T>&, hipStream_t);  \
  template void launch_linear_dz<T>(T*, float*, const T*, long, const T*,    \
                                    const ActParams&, long, int, hipStream_t);
INSTANTIATE(float)
INSTANTIATE(bf16)

}  // namespace gfa
