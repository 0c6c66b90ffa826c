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
// A row is held by L lanes, E elements each, as chunks of V elements (16
// bytes) that neighbouring lanes read side by side: L is a power of two up
// to 64 within a wave (several rows a wave where a row is short), or 256 or
// 1024 threads. x is read once and y written once. The loads need only the
// alignment of an element, so strides of any size take the same path.
//
// Widths that are no multiple of L * E (TAIL): a chunk that would end past
// the row is moved back to end with it. Its first elements then belong to
// the chunk before; they are computed and stored twice, alike, and left out
// of the sums. So no load or store is behind a branch, which would make the
// next row's loads wait (at 524288x96 bf16 the backward took 142 us with
// chunks read element by element at the end, 72 us this way).
template <typename T> struct Chunk;
template <> struct Chunk<float> {
  static constexpr int V = 4;
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Chunk<bf16> {
  static constexpr int V = 8;
  typedef u16 Vec __attribute__((ext_vector_type(8), aligned(2)));
};

template <typename T>
GFA_DEV typename Chunk<T>::Vec chunk_at(const T* p) {
  return *reinterpret_cast<const typename Chunk<T>::Vec*>(p);
}

// V parameters, whole chunks, from element i on; `none` for p null
template <int V, typename P>
GFA_DEV void params_at(float* v, const P* p, int i, float none) {
  constexpr int C = Chunk<P>::V;
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = none;
  if (!p) return;
#pragma unroll
  for (int k = 0; k < V; k += C) {
    const auto c = chunk_at(p + i + k);
#pragma unroll
    for (int j = 0; j < C; ++j) v[k + j] = raw_to_f32(c[j]);
  }
}

// A lane's part of a row: where its chunks begin, and which elements count.
// V is Chunk<T>::V, or 1 for rows shorter than a chunk.
template <typename T, int V, int E, bool TAIL>
struct Lane {
  using R = typename Raw<T>::type;
  int at[E / V], skip[E / V];  // skip: elements left out of the sums

  GFA_DEV Lane(int li, int L, int n) {
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
      const int i = (k * L + li) * V;
      at[k] = TAIL ? min(i, n - V) : i;
      skip[k] = TAIL ? i - at[k] : 0;
    }
  }
  GFA_DEV bool counts(int e) const { return !TAIL || e % V >= skip[e / V]; }
  GFA_DEV int index(int e) const { return at[e / V] + e % V; }

  GFA_DEV void load(R* v, const T* row) const {
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
      if constexpr (V == 1) {
        v[k] = reinterpret_cast<const R*>(row)[at[k]];
      } else {
        const auto c = chunk_at(row + at[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k * V + j] = c[j];
      }
    }
  }
  GFA_DEV void store(T* row, const float* v) const {
#pragma unroll
    for (int k = 0; k < E / V; ++k) {
      if constexpr (V == 1) {
        put(row + at[k], v[k]);
      } else {
        typename Chunk<T>::Vec c;
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = round_raw<T>(v[k * V + j]);
        *reinterpret_cast<typename Chunk<T>::Vec*>(row + at[k]) = c;
      }
    }
  }
  template <typename P>
  GFA_DEV void params(float* v, const P* p, float none) const {
#pragma unroll
    for (int k = 0; k < E / V; ++k)
      if constexpr (V == 1)
        v[k] = p ? to_f32(p[at[k]]) : none;
      else
        params_at<V>(v + k * V, p, at[k], none);
  }
};

template <typename T, typename P, int WAVES, int V, int E, bool TAIL>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256)
void layer_norm_fwd_rows(T* __restrict__ y, float* __restrict__ mean,
                         float* __restrict__ rstd, const T* __restrict__ x,
                         long x_stride, const P* __restrict__ w,
                         const P* __restrict__ b, long rows, int n, float eps,
                         int lanes) {
  // Blocks of 16 waves take one row each from a grid of all rows: the next
  // block's loads hide this one's barriers better than a row ahead does.
  constexpr bool kAhead = WAVES < 16;
  __shared__ float red[WAVES > 1 ? 4 * WAVES : 1];
  int turn = 0;
  const int L = WAVES == 1 ? lanes : WAVES * 64;
  const int li = threadIdx.x & (L - 1);
  const Lane<T, V, E, TAIL> lane(li, L, n);
  float wv[E], bv[E];
  lane.params(wv, w, 1.f);
  lane.params(bv, b, 0.f);
  // r0: the same for all lanes of a wave, which sum together
  const int own = threadIdx.x / L, per_block = blockDim.x / L;
  const long step = (long)gridDim.x * per_block;
  typename Raw<T>::type next[E];
  long r0 = (long)blockIdx.x * per_block;
  if (kAhead) lane.load(next, x + min(r0 + own, rows - 1) * x_stride);
  for (; r0 < rows; r0 += step) {
    const long r = r0 + own;
    const bool live = r < rows;
    if (!kAhead) lane.load(next, x + r * x_stride);
    float v[E];
    float s = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = raw_to_f32(next[e]);
      s += lane.counts(e) ? v[e] : 0.f;
    }
    // the next row is on its way while this one is summed and written
    if (kAhead && r0 + step < rows)
      lane.load(next, x + min(r + step, rows - 1) * x_stride);
    row_sum2<WAVES>(s, s2, lanes, red, turn);
    const float mu = s / n;
    s = s2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] -= mu;
      s += lane.counts(e) ? v[e] * v[e] : 0.f;
    }
    row_sum2<WAVES>(s, s2, lanes, red, turn);
    const float rs = 1.f / sqrtf(s / n + eps);
    if (!live) continue;
    if (li == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] * rs * wv[e] + bv[e];
    lane.store(y + r * n, v);
  }
}

// dw and db of eight columns from n0 on, all rows, by a block of its own
template <typename T, typename P, int THREADS>
GFA_DEV void layer_norm_columns(P* dw, P* db, const T* dy, long dy_stride,
                                const T* x, long x_stride, const float* mean,
                                const float* rstd, long rows, int n, int n0) {
  constexpr int Q = THREADS / 8;
  __shared__ float red[2][8][Q + 1];
  const int c = threadIdx.x & 7, q = threadIdx.x >> 3, i = n0 + c;
  float sw = 0.f, sb = 0.f;
  if (i < n) {
#pragma unroll 4
    for (long r = q; r < rows; r += Q) {
      const float d = to_f32(dy[r * dy_stride + i]);
      sw += d * (to_f32(x[r * x_stride + i]) - mean[r]) * rstd[r];
      sb += d;
    }
  }
  red[0][c][q] = sw;
  red[1][c][q] = sb;
  __syncthreads();
  if (threadIdx.x < 16) {
    const int k = threadIdx.x >> 3;
    P* out = k ? db : dw;
    if (!out || i >= n) return;
    float s = 0.f;
    for (int g = 0; g < Q; ++g) s += red[k][c][g];
    put(out + i, s);
  }
}

// One pass over x and dy: dx, and the block's sums over its rows of dy * xn
// and dy for the parameters, held in registers until the rows are through.
// Where the rows are few, blocks behind the first row_blocks make dw and db
// instead, from x and dy again: one launch where the sums of blocks take two.
template <typename T, typename P, int WAVES, int V, int E, bool TAIL>
__global__ __launch_bounds__(WAVES == 16 ? 1024 : 256)
void layer_norm_bwd_rows(T* __restrict__ dx, float* __restrict__ partial,
                         P* __restrict__ dw, P* __restrict__ db,
                         int row_blocks, const T* __restrict__ dy,
                         long dy_stride,
                         const T* __restrict__ x, long x_stride,
                         const P* __restrict__ w,
                         const float* __restrict__ mean,
                         const float* __restrict__ rstd, long rows, int n,
                         int lanes) {
  constexpr int kThreads = WAVES == 16 ? 1024 : 256;
  // a row ahead, except where its registers would spill
  constexpr bool kAhead = WAVES < 16 || E < 16;
  if ((int)blockIdx.x >= row_blocks) {
    layer_norm_columns<T, P, kThreads>(dw, db, dy, dy_stride, x, x_stride,
                                       mean, rstd, rows, n,
                                       (blockIdx.x - row_blocks) * 8);
    return;
  }
  __shared__ float red[WAVES > 1 ? 4 * WAVES : 1];
  // sums of the waves of a block, where they hold the same columns
  __shared__ float sums[WAVES == 1 ? kThreads * E : 1];
  int turn = 0;
  const int L = WAVES == 1 ? lanes : WAVES * 64;
  const int li = threadIdx.x & (L - 1);
  const int own = threadIdx.x / L, per_block = kThreads / L;
  const Lane<T, V, E, TAIL> lane(li, L, n);
  float wv[E], aw[E], ab[E];
  lane.params(wv, w, 1.f);
#pragma unroll
  for (int e = 0; e < E; ++e) aw[e] = ab[e] = 0.f;
  const long step = (long)row_blocks * per_block;
  typename Raw<T>::type next_x[E], next_d[E];
  float next_mu, next_rs;
  auto load = [&](long r) {
    const long at = min(r, rows - 1);
    lane.load(next_x, x + at * x_stride);
    lane.load(next_d, dy + at * dy_stride);
    next_mu = mean[at];
    next_rs = rstd[at];
  };
  long r0 = (long)blockIdx.x * per_block;
  if (kAhead) load(r0 + own);
  for (; r0 < rows; r0 += step) {
    const long r = r0 + own;
    const bool live = r < rows;
    if (!kAhead) load(r);
    const float mu = next_mu, rs = next_rs;
    float xn[E], d[E];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      xn[e] = raw_to_f32(next_x[e]);
      d[e] = raw_to_f32(next_d[e]);
    }
    if (kAhead && r0 + step < rows) load(r + step);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      xn[e] = (xn[e] - mu) * rs;
      if (live) {
        aw[e] += d[e] * xn[e];
        ab[e] += d[e];
      }
      d[e] *= wv[e];
      const float t = lane.counts(e) ? d[e] : 0.f;
      s1 += t;
      s2 += t * xn[e];
    }
    if (!dx) continue;
    row_sum2<WAVES>(s1, s2, lanes, red, turn);
    if (!live) continue;
    const float m1 = s1 / n, m2 = s2 / n;
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = rs * (d[e] - m1 - xn[e] * m2);
    lane.store(dx + r * n, d);
  }
  if (!partial) return;
  float* pw = partial + (long)blockIdx.x * n;
  float* pb = partial + ((long)row_blocks + blockIdx.x) * n;
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane.counts(e)) {
        pw[lane.index(e)] = aw[e];
        pb[lane.index(e)] = ab[e];
      }
  } else {
    // column i of the block's row group q is at sums[q * n + i]: n <= L * E
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (lane.counts(e)) sums[own * n + lane.index(e)] = k ? ab[e] : aw[e];
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        float s = 0.f;
        for (int q = 0; q < per_block; ++q) s += sums[q * n + i];
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

// sum over a block of 1024; every thread gets it
GFA_DEV float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += red[i];
  return s;
}

// f(i, chunk) for a thread's chunks of a row of n elements, then f1(i) for its
// elements behind the last whole chunk. Such a row is read again from the
// nearest cache that holds it: 1024 threads and whole chunks, since what
// bounds a block is how much it has under way (2048x32768 bf16: forward 72
// us, backward 168 us; 169 and 256 us with 256 threads and single elements).
template <int V, typename F, typename F1>
GFA_DEV void over_row(int n, F&& f, F1&& f1) {
  const int whole = n / V * V;
#pragma unroll 2
  for (int i = threadIdx.x * V; i < whole; i += 1024 * V) f(i);
  for (int i = whole + threadIdx.x; i < n; i += 1024) f1(i);
}
template <typename T, typename P>
__global__ __launch_bounds__(1024)
void layer_norm_fwd_kernel(T* __restrict__ y, float* __restrict__ mean,
                           float* __restrict__ rstd,
                           const T* __restrict__ x, long x_stride,
                           const P* __restrict__ w, const P* __restrict__ b,
                           long rows, int n, float eps) {
  constexpr int V = Chunk<T>::V;
  __shared__ float red[16];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    T* yr = y + r * n;
    float s = 0.f;
    over_row<V>(
        n,
        [&](int i) {
          const auto c = chunk_at(xr + i);
#pragma unroll
          for (int j = 0; j < V; ++j) s += raw_to_f32(c[j]);
        },
        [&](int i) { s += to_f32(xr[i]); });
    const float mu = block_sum(s, red) / n;
    float v = 0.f;
    auto square = [&](float a) { v += (a - mu) * (a - mu); };
    over_row<V>(
        n,
        [&](int i) {
          const auto c = chunk_at(xr + i);
#pragma unroll
          for (int j = 0; j < V; ++j) square(raw_to_f32(c[j]));
        },
        [&](int i) { square(to_f32(xr[i])); });
    const float rs = 1.f / sqrtf(block_sum(v, red) / n + eps);
    if (threadIdx.x == 0 && mean) {
      mean[r] = mu;
      rstd[r] = rs;
    }
    auto out = [&](float a, float wi, float bi) {
      return (a - mu) * rs * wi + bi;
    };
    over_row<V>(
        n,
        [&](int i) {
          const auto c = chunk_at(xr + i);
          float wv[V], bv[V];
          params_at<V>(wv, w, i, 1.f);
          params_at<V>(bv, b, i, 0.f);
          typename Chunk<T>::Vec o;
#pragma unroll
          for (int j = 0; j < V; ++j)
            o[j] = round_raw<T>(out(raw_to_f32(c[j]), wv[j], bv[j]));
          *reinterpret_cast<typename Chunk<T>::Vec*>(yr + i) = o;
        },
        [&](int i) {
          put(yr + i, out(to_f32(xr[i]), w ? to_f32(w[i]) : 1.f,
                          b ? to_f32(b[i]) : 0.f));
        });
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(1024)
void layer_norm_dx_kernel(T* __restrict__ dx, const T* __restrict__ dy,
                          long dy_stride, const T* __restrict__ x,
                          long x_stride, const P* __restrict__ w,
                          const float* __restrict__ mean,
                          const float* __restrict__ rstd, long rows, int n) {
  constexpr int V = Chunk<T>::V;
  __shared__ float red[16];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * x_stride;
    const T* dr = dy + r * dy_stride;
    T* out = dx + r * n;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    auto add = [&](float a, float g) {
      s1 += g;
      s2 += g * (a - mu) * rs;
    };
    over_row<V>(
        n,
        [&](int i) {
          const auto a = chunk_at(xr + i), d = chunk_at(dr + i);
          float wv[V];
          params_at<V>(wv, w, i, 1.f);
#pragma unroll
          for (int j = 0; j < V; ++j)
            add(raw_to_f32(a[j]), raw_to_f32(d[j]) * wv[j]);
        },
        [&](int i) {
          add(to_f32(xr[i]), to_f32(dr[i]) * (w ? to_f32(w[i]) : 1.f));
        });
    const float m1 = block_sum(s1, red) / n;
    const float m2 = block_sum(s2, red) / n;
    auto value = [&](float a, float g) {
      return rs * (g - m1 - (a - mu) * rs * m2);
    };
    over_row<V>(
        n,
        [&](int i) {
          const auto a = chunk_at(xr + i), d = chunk_at(dr + i);
          float wv[V];
          params_at<V>(wv, w, i, 1.f);
          typename Chunk<T>::Vec o;
#pragma unroll
          for (int j = 0; j < V; ++j)
            o[j] = round_raw<T>(
                value(raw_to_f32(a[j]), raw_to_f32(d[j]) * wv[j]));
          *reinterpret_cast<typename Chunk<T>::Vec*>(out + i) = o;
        },
        [&](int i) {
          put(out + i, value(to_f32(xr[i]),
                             to_f32(dr[i]) * (w ? to_f32(w[i]) : 1.f)));
        });
  }
}

// thread: a chunk of columns, the last moved back to end with the row;
// block: 256 chunks of one group of rows
template <typename T>
__global__ __launch_bounds__(256)
void layer_norm_dwb_kernel(float* __restrict__ partial,
                           const T* __restrict__ dy, long dy_stride,
                           const T* __restrict__ x, long x_stride,
                           const float* __restrict__ mean,
                           const float* __restrict__ rstd, long rows, int n) {
  constexpr int V = Chunk<T>::V;
  const int first = (blockIdx.x * 256 + threadIdx.x) * V;
  const int groups = gridDim.y;
  const long per = (rows + groups - 1) / groups;
  const long r0 = blockIdx.y * per, r1 = min(r0 + per, rows);
  if (first >= n) return;
  const int i = min(first, n - V);
  float sw[V] = {}, sb[V] = {};
#pragma unroll 2
  for (long r = r0; r < r1; ++r) {
    const auto a = chunk_at(x + r * x_stride + i);
    const auto d = chunk_at(dy + r * dy_stride + i);
    const float mu = mean[r], rs = rstd[r];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sw[j] += raw_to_f32(d[j]) * (raw_to_f32(a[j]) - mu) * rs;
      sb[j] += raw_to_f32(d[j]);
    }
  }
  float* pw = partial + (long)blockIdx.y * n + i;
  float* pb = partial + (long)(groups + blockIdx.y) * n + i;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    pw[j] = sw[j];
    pb[j] = sb[j];
  }
}

// out[k][i] = scale * sum_g partial[k][g][i] for k of grid y: 32 columns a
// block and 32 threads a column, four of whose loads are on their way at a
// time (one after the other, 1024 groups took 40 us).
template <typename P>
__global__ __launch_bounds__(1024)
void sum_groups_kernel(P* __restrict__ out0, P* __restrict__ out1,
                       const float* __restrict__ partial, int groups, int n,
                       float scale) {
  __shared__ float red[32][33];
  P* out = blockIdx.y ? out1 : out0;
  if (!out) return;
  partial += (long)blockIdx.y * groups * n;
  const int c = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + c;
  float s = 0.f;
  if (i < n)
    for (int g = q; g < groups; g += 128) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = g + 32 * k < groups ? partial[(long)(g + 32 * k) * n + i] : 0.f;
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  red[q][c] = s;
  __syncthreads();
  // the 32 sums of a column, side by side in half a wave
  s = red[c][q];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor(s, o, 32);
  const int col = blockIdx.x * 32 + q;
  if (c == 0 && col < n) put(out + col, s * scale);
}

template <typename P>
void launch_sum_groups(P* out0, P* out1, const float* partial, int groups,
                       int n, float scale, hipStream_t s) {
  hipLaunchKernelGGL(sum_groups_kernel<P>, dim3(ceil_div(n, 32), out1 ? 2 : 1),
                     dim3(1024), 0, s, out0, out1, partial, groups, n, scale);
}

namespace {

// How a row of n elements of type T is held: `waves` of a block (1, 4, 16; 0:
// too wide for registers), `lanes` of one wave, `v` elements a chunk and `e`
// a lane.
struct RowPlan {
  int waves, lanes, v, e, per_block;
  bool tail;
};

// most4: elements a lane of a block of 4 waves may hold
template <typename T>
RowPlan row_plan(int n, int most4 = 16) {
  RowPlan p{0, 64, Chunk<T>::V, 16, 1, true};
  if (n < p.v) p.v = 1;
  for (int waves : {1, 4, 16})
    if (!p.waves && n <= waves * 64 * (waves == 4 ? most4 : 16))
      p.waves = waves;
  if (!p.waves) return p;
  p.e = p.v;
  while (n > p.waves * 64 * p.e) p.e *= 2;
  if (p.waves == 1) {
    while (p.lanes > 1 && n <= p.lanes / 2 * p.v) p.lanes /= 2;
    p.per_block = 256 / p.lanes;
  }
  p.tail = n != (p.waves == 1 ? p.lanes : p.waves * 64) * p.e;
  return p;
}

template <int N> using Int = std::integral_constant<int, N>;

// f(waves, v, e, tail) with all four as compile-time constants
template <typename T, bool FWD, typename F>
void with_plan(const RowPlan& p, F&& f) {
  constexpr int V = Chunk<T>::V;
  auto with_e = [&](auto waves, auto tail) {
    if (p.e == V) return f(waves, Int<V>{}, Int<V>{}, tail);
    if (p.e == 2 * V) return f(waves, Int<V>{}, Int<2 * V>{}, tail);
    if constexpr (V == 4 || (FWD && waves() == 4))
      f(waves, Int<V>{}, Int<4 * V>{}, tail);
  };
  auto with_tail = [&](auto waves) {
    if (p.tail) return with_e(waves, std::true_type{});
    with_e(waves, std::false_type{});
  };
  if (p.v == 1) return f(Int<1>{}, Int<1>{}, Int<1>{}, std::true_type{});
  if (p.waves == 1) return with_tail(Int<1>{});
  if (p.waves == 4) return with_tail(Int<4>{});
  with_tail(Int<16>{});
}

}  // namespace

template <typename T, typename P>
void launch_layer_norm_fwd(T* y, float* mean, float* rstd, const T* x,
                           long x_stride, const P* w, const P* b, long rows,
                           int n, float eps, hipStream_t s) {
  // bf16 rows up to 8192 stay in 4 waves (8192x8192: 16 waves 79 us)
  const RowPlan p = row_plan<T>(n, sizeof(T) == 2 ? 32 : 16);
  if (!p.waves) {
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, P>), dim3(grid), dim3(1024),
                       0, s, y, mean, rstd, x, x_stride, w, b, rows, n, eps);
    return;
  }
  const long blocks = (rows + p.per_block - 1) / p.per_block;
  const long most = p.waves == 16 ? 1 << 20 : 1536;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  with_plan<T, true>(p, [&](auto waves, auto v, auto e, auto tail) {
    hipLaunchKernelGGL(
        (layer_norm_fwd_rows<T, P, waves(), v(), e(), tail()>), dim3(grid),
        dim3(waves() == 16 ? 1024 : 256), 0, s, y, mean, rstd, x, x_stride, w,
        b, rows, n, eps, p.lanes);
  });
}

int layer_norm_bwd_groups(long rows, int n, bool f32) {
  const RowPlan p = f32 ? row_plan<float>(n) : row_plan<bf16>(n);
  if (!p.waves) {
    const long g = (rows + 63) / 64;
    return (int)(g < 256 ? g : 256);
  }
  const long blocks = (rows + p.per_block - 1) / p.per_block;
  // two blocks a CU (one of 16 waves), each a row ahead, keep the memory
  // busy; more only add sums to be read again (131072x512 bf16: 80 us with
  // 512, 82 us with 1024, 91 us with 1536)
  const long most = p.waves == 16 ? 256 : 512;
  return (int)(blocks < most ? blocks : most);
}

// Whether dw and db go by sums of blocks: not where x and dy are so small that
// reading them again, eight columns a block, is less than a launch.
bool layer_norm_bwd_sums(long rows, int n, bool f32) {
  const RowPlan p = f32 ? row_plan<float>(n) : row_plan<bf16>(n);
  return rows > 1024 || rows * n > 1 << 21 || !p.waves;
}

template <typename T, typename P>
void launch_layer_norm_bwd(T* dx, P* dw, P* db, float* partial, const T* dy,
                           long dy_stride, const T* x, long x_stride,
                           const P* w, const float* mean, const float* rstd,
                           long rows, int n, hipStream_t s) {
  const RowPlan p = row_plan<T>(n);
  const int groups = layer_norm_bwd_groups(rows, n, sizeof(T) == 4);
  const bool columns = !partial && (dw || db);
  if (p.waves) {
    const int blocks = (dx || partial ? groups : 0);
    const int grid = blocks + (columns ? ceil_div(n, 8) : 0);
    with_plan<T, false>(p, [&](auto waves, auto v, auto e, auto tail) {
      hipLaunchKernelGGL(
          (layer_norm_bwd_rows<T, P, waves(), v(), e(), tail()>), dim3(grid),
          dim3(waves() == 16 ? 1024 : 256), 0, s, dx, partial, dw, db, blocks,
          dy, dy_stride, x, x_stride, w, mean, rstd, rows, n, p.lanes);
    });
  } else {
    if (dx) {
      const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
      hipLaunchKernelGGL((layer_norm_dx_kernel<T, P>), dim3(grid), dim3(1024),
                         0, s, dx, dy, dy_stride, x, x_stride, w, mean, rstd,
                         rows, n);
    }
    if (partial)
      hipLaunchKernelGGL(layer_norm_dwb_kernel<T>,
                         dim3(ceil_div(n, 256 * Chunk<T>::V), groups),
                         dim3(256), 0, s, partial, dy, dy_stride, x, x_stride,
                         mean, rstd, rows, n);
  }
  if (partial)
    launch_sum_groups<P>(dw, db, partial, groups, n, 1.f, s);
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
template void launch_sum_groups<float>(float*, float*, const float*, int, int,
                                       float, hipStream_t);
template void launch_sum_groups<bf16>(bf16*, bf16*, const float*, int, int,
                                      float, hipStream_t);

}  // namespace gfa
