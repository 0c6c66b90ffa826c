// Layer norm over the last dimension for gfx950.
//
//   xn = (x - mean) * rstd,  y = xn * w + b
//   g  = dy * w
//   dx = rstd * (g - mean_n(g) - xn * mean_n(g * xn))
//   dw = sum_rows dy * xn,   db = sum_rows dy
//
// Statistics and sums in float; the variance from the centred values, so a
// mean far from zero costs no digits.
#include <type_traits>

#include "rows.h"

namespace gfa {

// ---- sums over lanes ----
// Data-parallel moves within 16 lanes and the two half-exchanges of gfx950:
// no trip through LDS, which a shuffle would take.
template <int CTRL>
GFA_DEV float dpp(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xf, 0xf,
                                  true));
}

// sum over aligned groups of `lanes` (a power of two up to 64); every lane
// of a group gets it. After the first two steps all four lanes of a quad are
// alike, so a mirror does what an exchange would.
GFA_DEV float group_sum(float v, int lanes) {
  if (lanes > 1) v += dpp<0xB1>(v);   // lane ^ 1
  if (lanes > 2) v += dpp<0x4E>(v);   // lane ^ 2
  if (lanes > 4) v += dpp<0x141>(v);  // mirrored within 8
  if (lanes > 8) v += dpp<0x140>(v);  // mirrored within 16
  if (lanes > 16) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lanes > 32) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// sums of a and b over WAVES waves (one row); red has 2 * 2 * WAVES floats,
// its halves used in turn (`turn` flips) so that one barrier is enough
template <int WAVES>
GFA_DEV void row_sum2(float& a, float& b, int lanes, float* red, int& turn) {
  a = group_sum(a, WAVES == 1 ? lanes : 64);
  b = group_sum(b, WAVES == 1 ? lanes : 64);
  if constexpr (WAVES > 1) {
    float* r = red + turn * 2 * WAVES;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
      r[threadIdx.x >> 6] = a;
      r[WAVES + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      a += r[i];
      b += r[WAVES + i];
    }
  }
}

// ---- rows in registers ----
// A row is held by L lanes, E elements each, as chunks of 16 bytes that
// neighbouring lanes read side by side: L is a power of two up to 64 within
// a wave (several rows a wave where a row is short), or 256 or 1024 threads.
// x is read once and y written once; the loads need only the alignment of
// an element, so strides and widths of any size take the same path, with
// the last, partial chunk read element by element.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int V = 4;
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Chunk<bf16> {
  static constexpr int V = 8;
  typedef u16 Vec __attribute__((ext_vector_type(8), aligned(2)));
};

// v[0..V) = p[i..i+V), zero from n on
template <typename T>
GFA_DEV void load_chunk(float* v, const T* p, int i, int n) {
  using C = Chunk<T>;
  if (i + C::V <= n) {
    const auto c = *reinterpret_cast<const typename C::Vec*>(p + i);
#pragma unroll
    for (int j = 0; j < C::V; ++j) v[j] = raw_to_f32(c[j]);
  } else {
#pragma unroll
    for (int j = 0; j < C::V; ++j) v[j] = i + j < n ? to_f32(p[i + j]) : 0.f;
  }
}

template <typename T>
GFA_DEV void store_chunk(T* p, const float* v, int i, int n) {
  using C = Chunk<T>;
  if (i + C::V <= n) {
    typename C::Vec c;
#pragma unroll
    for (int j = 0; j < C::V; ++j)
      c[j] = round_raw<T>(v[j]);
    *reinterpret_cast<typename C::Vec*>(p + i) = c;
  } else {
#pragma unroll
    for (int j = 0; j < C::V; ++j)
      if (i + j < n) put(p + i + j, v[j]);
  }
}

// V parameters of type P, `none` where there are none or from n on
template <int V, typename P>
GFA_DEV void load_params(float* v, const P* p, int i, int n, float none) {
#pragma unroll
  for (int j = 0; j < V; ++j)
    v[j] = p && i + j < n ? to_f32(p[i + j]) : none;
}

template <typename T, typename P, int WAVES, int E>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256)
void layer_norm_fwd_rows(T* __restrict__ y, float* __restrict__ mean,
                         float* __restrict__ rstd, const T* __restrict__ x,
                         long x_stride, const P* __restrict__ w,
                         const P* __restrict__ b, long rows, int n, float eps,
                         int lanes) {
  constexpr int V = Chunk<T>::V;
  __shared__ float red[WAVES > 1 ? 4 * WAVES : 1];
  int turn = 0;
  const int L = WAVES == 1 ? lanes : WAVES * 64;
  const int li = threadIdx.x & (L - 1);
  const int per_block = blockDim.x / L;
  float wv[E], bv[E];
#pragma unroll
  for (int c = 0; c < E; c += V) {
    load_params<V>(wv + c, w, c * L + li * V, n, 1.f);
    load_params<V>(bv + c, b, c * L + li * V, n, 0.f);
  }
  // r0: the same for all lanes of a wave, which sum together
  const int own = threadIdx.x / L;
  for (long r0 = (long)blockIdx.x * per_block; r0 < rows;
       r0 += (long)gridDim.x * per_block) {
    const long r = r0 + own;
    const bool live = r < rows;
    const T* xr = x + (live ? r : r0) * x_stride;
    float v[E];
    float s = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < E; c += V) {
      load_chunk<T>(v + c, xr, c * L + li * V, n);
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[c + j];
    }
    row_sum2<WAVES>(s, s2, lanes, red, turn);
    const float mu = s / n;
    s = s2 = 0.f;
#pragma unroll
    for (int c = 0; c < E; c += V) {
      const int left = n - (c * L + li * V);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[c + j] -= mu;
        s += j < left ? v[c + j] * v[c + j] : 0.f;
      }
    }
    row_sum2<WAVES>(s, s2, lanes, red, turn);
    const float rs = 1.f / sqrtf(s / n + eps);
    if (!live) continue;
    if (li == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
#pragma unroll
    for (int c = 0; c < E; c += V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        v[c + j] = v[c + j] * rs * wv[c + j] + bv[c + j];
      store_chunk<T>(y + r * n, v + c, c * L + li * V, n);
    }
  }
}

// One pass over x and dy: dx, and the block's sums over its rows of dy * xn
// and dy for the parameters, held in registers until the rows are through.
template <typename T, typename P, int WAVES, int E>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256)
void layer_norm_bwd_rows(T* __restrict__ dx, float* __restrict__ partial,
                         const T* __restrict__ dy, long dy_stride,
                         const T* __restrict__ x, long x_stride,
                         const P* __restrict__ w,
                         const float* __restrict__ mean,
                         const float* __restrict__ rstd, long rows, int n,
                         int lanes) {
  constexpr int V = Chunk<T>::V;
  constexpr int kThreads = WAVES == 16 ? 1024 : 256;
  __shared__ float red[WAVES > 1 ? 4 * WAVES : 1];
  // sums of the waves of a block, where they hold the same columns
  __shared__ float sums[WAVES == 1 ? kThreads * E : 1];
  int turn = 0;
  const int L = WAVES == 1 ? lanes : WAVES * 64;
  const int li = threadIdx.x & (L - 1);
  const int per_block = kThreads / L;
  const int own = threadIdx.x / L;
  float wv[E], aw[E], ab[E];
#pragma unroll
  for (int c = 0; c < E; c += V)
    load_params<V>(wv + c, w, c * L + li * V, n, 1.f);
#pragma unroll
  for (int c = 0; c < E; ++c) aw[c] = ab[c] = 0.f;
  for (long r0 = (long)blockIdx.x * per_block; r0 < rows;
       r0 += (long)gridDim.x * per_block) {
    const long r = r0 + own;
    const bool live = r < rows;
    const long at = live ? r : r0;
    const float mu = mean[at], rs = rstd[at];
    float xn[E], d[E];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int c = 0; c < E; c += V) {
      load_chunk<T>(xn + c, x + at * x_stride, c * L + li * V, n);
      load_chunk<T>(d + c, dy + at * dy_stride, c * L + li * V, n);
    }
    if (!live) {
#pragma unroll
      for (int c = 0; c < E; ++c) d[c] = xn[c] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < E; ++c) {
      xn[c] = (xn[c] - mu) * rs;
      if (live) {
        aw[c] += d[c] * xn[c];
        ab[c] += d[c];
      }
      d[c] *= wv[c];
      s1 += d[c];
      s2 += d[c] * xn[c];
    }
    if (!dx) continue;
    row_sum2<WAVES>(s1, s2, lanes, red, turn);
    if (!live) continue;
    const float m1 = s1 / n, m2 = s2 / n;
#pragma unroll
    for (int c = 0; c < E; c += V) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        d[c + j] = rs * (d[c + j] - m1 - xn[c + j] * m2);
      store_chunk<T>(dx + r * n, d + c, c * L + li * V, n);
    }
  }
  if (!partial) return;
  float* pw = partial + (long)blockIdx.x * n;
  float* pb = partial + ((long)gridDim.x + blockIdx.x) * n;
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int c = 0; c < E; c += V) {
#pragma unroll
      for (int h = 0; h < V; h += 4) {
        store_chunk<float>(pw, aw + c + h, c * L + li * V + h, n);
        store_chunk<float>(pb, ab + c + h, c * L + li * V + h, n);
      }
    }
  } else {
    // column i of the block's row group q is at sums[q * width + i]
    const int width = L * E;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < E; c += V)
#pragma unroll
        for (int j = 0; j < V; ++j)
          sums[own * width + c * L + li * V + j] = k ? ab[c + j] : aw[c + j];
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        float s = 0.f;
        for (int q = 0; q < per_block; ++q) s += sums[q * width + i];
        (k ? pb : pw)[i] = s;
      }
    }
  }
}

// ---- rows of any width ----

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
      put(y + r * n + i, o);
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
      put(dx + r * n + i, rs * (g - m1 - xn * m2));
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

// out[i] = scale * sum_g partial[g][i]: 32 columns a block, 8 threads a
// column, each of which takes every 8th group
template <typename P>
__global__ __launch_bounds__(256)
void sum_groups_kernel(P* __restrict__ out, const float* __restrict__ partial,
                       int groups, int n, float scale) {
  __shared__ float red[8][33];
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + c;
  float s = 0.f;
  if (i < n)
    for (int g = q; g < groups; g += 8) s += partial[(long)g * n + i];
  red[q][c] = s;
  __syncthreads();
  if (q == 0 && i < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][c];
    put(out + i, s * scale);
  }
}

template <typename P>
void launch_sum_groups(P* out, const float* partial, int groups, int n,
                       float scale, hipStream_t s) {
  hipLaunchKernelGGL(sum_groups_kernel<P>, dim3(ceil_div(n, 32)), dim3(256),
                     0, s, out, partial, groups, n, scale);
}

namespace {

// How a row of n elements of type T is held: `waves` of a block (1, 4, 16; 0:
// too wide for registers), `lanes` of one wave, `e` elements a lane.
struct RowPlan {
  int waves, lanes, e, per_block;
};

template <typename T>
RowPlan row_plan(int n) {
  const int v = Chunk<T>::V;
  RowPlan p{0, 64, 16, 1};
  for (int waves : {1, 4, 16})
    if (!p.waves && n <= waves * 64 * 16) p.waves = waves;
  if (!p.waves) return p;
  p.e = v;
  while (n > p.waves * 64 * p.e) p.e *= 2;
  if (p.waves == 1) {
    while (p.lanes > 1 && n <= p.lanes / 2 * v) p.lanes /= 2;
    p.per_block = 256 / p.lanes;
  }
  return p;
}

// f(waves, e) with both as compile-time constants
template <typename T, typename F>
void with_plan(const RowPlan& p, F&& f) {
  auto with_e = [&](auto waves) {
    if constexpr (Chunk<T>::V == 4)
      if (p.e == 4) return f(waves, std::integral_constant<int, 4>{});
    if (p.e == 8) return f(waves, std::integral_constant<int, 8>{});
    f(waves, std::integral_constant<int, 16>{});
  };
  if (p.waves == 1) return with_e(std::integral_constant<int, 1>{});
  if (p.waves == 4) return with_e(std::integral_constant<int, 4>{});
  with_e(std::integral_constant<int, 16>{});
}

}  // namespace

template <typename T, typename P>
void launch_layer_norm_fwd(T* y, float* mean, float* rstd, const T* x,
                           long x_stride, const P* w, const P* b, long rows,
                           int n, float eps, hipStream_t s) {
  const RowPlan p = row_plan<T>(n);
  if (!p.waves) {
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P>), dim3(grid), dim3(256),
                       0, s, y, mean, rstd, x, x_stride, w, b, rows, n, eps);
    return;
  }
  const long blocks = (rows + p.per_block - 1) / p.per_block;
  const long most = p.waves == 16 ? 512 : 2048;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  with_plan<T>(p, [&](auto waves, auto e) {
    hipLaunchKernelGGL((layer_norm_fwd_rows<T, P, waves(), e()>), dim3(grid),
                       dim3(p.waves == 16 ? 1024 : 256), 0, s, y, mean, rstd,
                       x, x_stride, w, b, rows, n, eps, p.lanes);
  });
}

int layer_norm_bwd_groups(long rows, int n, bool f32) {
  const RowPlan p = f32 ? row_plan<float>(n) : row_plan<bf16>(n);
  if (!p.waves) {
    const long g = (rows + 63) / 64;
    return (int)(g < 256 ? g : 256);
  }
  const long blocks = (rows + p.per_block - 1) / p.per_block;
  const long most = p.waves == 16 ? 512 : 1024;
  return (int)(blocks < most ? blocks : most);
}

template <typename T, typename P>
void launch_layer_norm_bwd(T* dx, P* dw, P* db, float* partial, const T* dy,
                           long dy_stride, const T* x, long x_stride,
                           const P* w, const float* mean, const float* rstd,
                           long rows, int n, hipStream_t s) {
  const RowPlan p = row_plan<T>(n);
  const int groups = layer_norm_bwd_groups(rows, n, sizeof(T) == 4);
  if (p.waves) {
    with_plan<T>(p, [&](auto waves, auto e) {
      hipLaunchKernelGGL((layer_norm_bwd_rows<T, P, waves(), e()>),
                         dim3(groups), dim3(p.waves == 16 ? 1024 : 256), 0, s,
                         dx, partial, dy, dy_stride, x, x_stride, w, mean,
                         rstd, rows, n, p.lanes);
    });
  } else {
    if (dx) {
      const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
      hipLaunchKernelGGL((layer_norm_dx_kernel<T, P>), dim3(grid), dim3(256),
                         0, s, dx, dy, dy_stride, x, x_stride, w, mean, rstd,
                         rows, n);
    }
    if (partial)
      hipLaunchKernelGGL(layer_norm_dwb_kernel<T>,
                         dim3(ceil_div(n, 256), groups), dim3(256), 0, s,
                         partial, dy, dy_stride, x, x_stride, mean, rstd,
                         rows, n);
  }
  if (dw) launch_sum_groups<P>(dw, partial, groups, n, 1.f, s);
  if (db)
    launch_sum_groups<P>(db, partial + (long)groups * n, groups, n, 1.f, s);
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
