// Layer norm over the last dimension for gfx950.
//
//   xn = (x - mean) * rstd,  y = xn * w + b
//   g  = dy * w
//   dx = rstd * (g - mean_n(g) - xn * mean_n(g * xn))
//   dw = sum_rows dy * xn,   db = sum_rows dy
//
// Statistics and sums in float; the variance from the centred values, so a
// mean far from zero costs no digits.
#include "rows.h"

namespace gfa {

GFA_DEV float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// sum over a block of 256; every thread gets it
GFA_DEV float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

template <typename T, typename P>
__global__ __launch_bounds__(256)
void layer_norm_fwd_kernel(T* __restrict__ y, float* __restrict__ mean,
                           float* __restrict__ rstd,
                           const T* __restrict__ x, long x_stride,
                           const P* __restrict__ w, const P* __restrict__ b,
                           long rows, int n, float eps) {
  __shared__ float red[4];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    float s = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) s += to_f32(xr[i]);
    const float mu = block_sum(s, red) / n;
    float v = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float d = to_f32(xr[i]) - mu;
      v += d * d;
    }
    const float rs = 1.f / sqrtf(block_sum(v, red) / n + eps);
    if (threadIdx.x == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
    for (int i = threadIdx.x; i < n; i += 256) {
      float o = (to_f32(xr[i]) - mu) * rs;
      if (w) o *= to_f32(w[i]);
      if (b) o += to_f32(b[i]);
      y[r * n + i] = from_f32<T>(o);
    }
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(256)
void layer_norm_dx_kernel(T* __restrict__ dx, const T* __restrict__ dy,
                          long dy_stride, const T* __restrict__ x,
                          long x_stride, const P* __restrict__ w,
                          const float* __restrict__ mean,
                          const float* __restrict__ rstd, long rows, int n) {
  __shared__ float red[4];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    const T* dr = dy + r * dy_stride;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float g = to_f32(dr[i]) * (w ? to_f32(w[i]) : 1.f);
      s1 += g;
      s2 += g * (to_f32(xr[i]) - mu) * rs;
    }
    const float m1 = block_sum(s1, red) / n;
    const float m2 = block_sum(s2, red) / n;
    for (int i = threadIdx.x; i < n; i += 256) {
      const float g = to_f32(dr[i]) * (w ? to_f32(w[i]) : 1.f);
      const float xn = (to_f32(xr[i]) - mu) * rs;
      dx[r * n + i] = from_f32<T>(rs * (g - m1 - xn * m2));
    }
  }
}

// thread: one column; block: 256 columns of one group of rows
template <typename T>
__global__ __launch_bounds__(256)
void layer_norm_dwb_kernel(float* __restrict__ partial,
                           const T* __restrict__ dy, long dy_stride,
                           const T* __restrict__ x, long x_stride,
                           const float* __restrict__ mean,
                           const float* __restrict__ rstd, long rows, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int groups = gridDim.y;
  const long per = (rows + groups - 1) / groups;
  const long r0 = blockIdx.y * per, r1 = min(r0 + per, rows);
  if (i >= n) return;
  float sw = 0.f, sb = 0.f;
  for (long r = r0; r < r1; ++r) {
    const float d = to_f32(dy[r * dy_stride + i]);
    sw += d * (to_f32(x[r * x_stride + i]) - mean[r]) * rstd[r];
    sb += d;
  }
  partial[(long)blockIdx.y * n + i] = sw;
  partial[(long)(groups + blockIdx.y) * n + i] = sb;
}

template <typename P>
__global__ __launch_bounds__(256)
void sum_groups_kernel(P* __restrict__ out, const float* __restrict__ partial,
                       int groups, int n, float scale) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int g = 0; g < groups; ++g) s += partial[(long)g * n + i];
  out[i] = from_f32<P>(s * scale);
}

template <typename P>
void launch_sum_groups(P* out, const float* partial, int groups, int n,
                       float scale, hipStream_t s) {
  hipLaunchKernelGGL(sum_groups_kernel<P>, dim3(ceil_div(n, 256)), dim3(256),
                     0, s, out, partial, groups, n, scale);
}

template <typename T, typename P>
void launch_layer_norm_fwd(T* y, float* mean, float* rstd, const T* x,
                           long x_stride, const P* w, const P* b, long rows,
                           int n, float eps, hipStream_t s) {
  const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
  hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P>), dim3(grid), dim3(256), 0,
                     s, y, mean, rstd, x, x_stride, w, b, rows, n, eps);
}

int layer_norm_bwd_groups(long rows, int n) {
  const long g = (rows + 63) / 64;
  return (int)(g < 256 ? g : 256);
}

template <typename T, typename P>
void launch_layer_norm_bwd(T* dx, P* dw, P* db, float* partial, const T* dy,
                           long dy_stride, const T* x, long x_stride,
                           const P* w, const float* mean, const float* rstd,
                           long rows, int n, hipStream_t s) {
  if (dx) {
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
    hipLaunchKernelGGL((layer_norm_dx_kernel<T, P>), dim3(grid), dim3(256), 0,
                       s, dx, dy, dy_stride, x, x_stride, w, mean, rstd, rows,
                       n);
  }
  if (dw || db) {
    const int groups = layer_norm_bwd_groups(rows, n);
    hipLaunchKernelGGL(layer_norm_dwb_kernel<T>,
                       dim3(ceil_div(n, 256), groups), dim3(256), 0, s,
                       partial, dy, dy_stride, x, x_stride, mean, rstd, rows,
                       n);
    if (dw) launch_sum_groups<P>(dw, partial, groups, n, 1.f, s);
    if (db)
      launch_sum_groups<P>(db, partial + (long)groups * n, groups, n, 1.f, s);
  }
}

#define INSTANTIATE(T, P)                                                     \
  template void launch_layer_norm_fwd<T, P>(T*, float*, float*, const T*,     \
                                            long, const P*, const P*, long,   \
                                            int, float, hipStream_t);         \
  template void launch_layer_norm_bwd<T, P>(                                  \
      T*, P*, P*, float*, const T*, long, const T*, long, const P*,           \
      const float*, const float*, long, int, hipStream_t);
INSTANTIATE(float, float)
INSTANTIATE(bf16, float)
INSTANTIATE(bf16, bf16)
template void launch_sum_groups<float>(float*, const float*, int, int, float,
                                       hipStream_t);
template void launch_sum_groups<bf16>(bf16*, const float*, int, int, float,
                                      hipStream_t);

}  // namespace gfa
