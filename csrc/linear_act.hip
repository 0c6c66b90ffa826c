// Matrix product with bias, activation and residual in its epilogue, and
// the products of its backward, for gfx950.
//
//   z  = alpha * A B^T + bias_gain * bias
//   y  = clamp(act(z) * gain) + residual
//   dz = dy * slope(z);  dx = dz W;  dW = dz^T x;  db = sum_rows dz
//
// A bf16 dz is kept as two bf16 numbers, and dx and dW are the sums of the
// products of both: rounded to one, dz would put as much error into dx and dW
// as their own rounding does.
//
// Every product is one C[m, n] = sum_k A[m, k] B[n, k] over operands that are
// contiguous along k ("rows") or along m or n ("columns"). Sums in float on
// the matrix cores; what leaves a kernel is rounded to T once.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "rows.h"

namespace gfa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
using LdsPtr = __attribute__((address_space(3))) void*;

// ---- tiles ----
// A block computes BM x BN of C with WM x WN waves. Both operands of a k-tile
// go from memory to LDS without passing through registers, 1 KB a wave and
// instruction; a k-tile is 128 bytes deep (64 bf16, 32 float) and two of them
// are in LDS, one being used while the other is filled, with one barrier a
// k-tile. Reads outside the operands return zero (the bounds are those of
// the buffer descriptor), so any M, N, K take this path as long as rows are
// 16-byte aligned.
//
// What bounds it: float the matrix cores (busy 94% of the time at 4096^3, 146
// TFLOP/s); bf16 8192x4096x4096 keeps them busy 67% (1175 TFLOP/s; dx 74%, dw
// 78%; a copy of the operands and the result would take 32 us); a short k
// leaves a tile's 128 KB of results, half of its 23 us at k = 512.
//
// LDS layout. Rows: [m][128 bytes], 16-byte granule g of row r at g ^ (r/2
// mod 8), so that the 16 rows a fragment read touches spread over all 64
// banks (conflicts: 2% of the LDS's busy cycles). Columns: [k][BX], granules
// of row k exchanged likewise; bf16 fragments come out of it through the
// transposing LDS read.
template <typename T, int BX, bool COLS>
struct Operand {
  static constexpr int ES = sizeof(T);
  static constexpr int BK = 128 / ES;
  static constexpr int kBytes = BX * 128;
  static constexpr int kGran = COLS ? BX * ES / 16 : 8;  // granules of a row

  // the granule of global memory that belongs at position p of LDS row r
  GFA_DEV static int swizzle(int r) {
    if (!COLS) return (r >> 1) & 7;
    // the rows that one fragment read touches: bf16 r mod 4 and r/8 mod 2,
    // float r/4 mod 4
    const int s = ES == 2 ? 2 * ((r & 3) | ((r >> 1) & 4)) : 4 * ((r >> 2) & 3);
    return s & (kGran - 1);
  }

  // byte offset from the tile's corner of what belongs at granule idx
  GFA_DEV static int source(int idx, int stride) {
    const int r = idx / kGran, p = idx % kGran;
    return r * stride * ES + ((p ^ swizzle(r)) << 4);
  }
};

// fragments of 16 (m or n) x 128 bits of k: what one lane gives to the
// matrix cores for a step of kStep
template <typename T> struct Unaligned;
template <> struct Unaligned<float> {
  typedef float Vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Unaligned<bf16> {
  typedef short Vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <typename T> struct Frag;
template <> struct Frag<bf16> {
  static constexpr int kStep = 32, kMfmas = 1, kColReads = 2;
  using Type = s16x8;
  template <int BX, bool COLS>
  GFA_DEV static Type read(const char* lds, int row0, int step, int lane) {
    using O = Operand<bf16, BX, COLS>;
    if constexpr (!COLS) {
      const int r = row0 + (lane & 15);
      const int g = step * 4 + (lane >> 4);
      return *reinterpret_cast<const Type*>(lds + r * 128 +
                                            ((g ^ O::swizzle(r)) << 4));
    } else {
      // four k of 16 columns each: lane i of 16 points at four columns of
      // row i / 4 and gets the four rows of column i
      s16x4 h[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int k = step * 32 + (lane >> 4) * 8 + q * 4 + ((lane & 15) >> 2);
        const int c = row0 + 4 * (lane & 3);
        h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(
                lds + k * (BX * 2) + (((c >> 3) ^ O::swizzle(k)) << 4) +
                (c & 7) * 2));
      }
      return Type{h[0][0], h[0][1], h[0][2], h[0][3],
                  h[1][0], h[1][1], h[1][2], h[1][3]};
    }
  }
  GFA_DEV static f32x4 mma(Type a, Type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
  }
};
template <> struct Frag<float> {
  // k = 4 * (lane / 16) + j in step j of 4
  static constexpr int kStep = 16, kMfmas = 4, kColReads = 4;
  using Type = f32x4;
  template <int BX, bool COLS>
  GFA_DEV static Type read(const char* lds, int row0, int step, int lane) {
    using O = Operand<float, BX, COLS>;
    if constexpr (!COLS) {
      const int r = row0 + (lane & 15);
      const int g = step * 4 + (lane >> 4);
      return *reinterpret_cast<const Type*>(lds + r * 128 +
                                            ((g ^ O::swizzle(r)) << 4));
    } else {
      Type v;
      const int c = row0 + (lane & 15);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = step * 16 + (lane >> 4) * 4 + j;
        v[j] = *reinterpret_cast<const float*>(
            lds + k * (BX * 4) + (((c >> 2) ^ O::swizzle(k)) << 4) +
            (c & 3) * 4);
      }
      return v;
    }
  }
  GFA_DEV static f32x4 mma(Type a, Type b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// Eight values of a row, at any alignment, as they are stored; zero from
// `left` on. Kept so until they are used: a conversion would wait for them.
template <typename T> struct Eight;
template <> struct Eight<float> {
  typedef float Half __attribute__((ext_vector_type(4), aligned(4)));
  Half a, b;
  GFA_DEV float operator[](int j) const { return j < 4 ? a[j] : b[j - 4]; }
  GFA_DEV void load(const float* p) {
    a = *reinterpret_cast<const Half*>(p);
    b = *reinterpret_cast<const Half*>(p + 4);
  }
  GFA_DEV void load(const float* p, int left) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = j < left ? p[j] : 0.f;
      b[j] = j + 4 < left ? p[j + 4] : 0.f;
    }
  }
};
template <> struct Eight<bf16> {
  typedef u16 Vec __attribute__((ext_vector_type(8), aligned(2)));
  Vec a;
  GFA_DEV float operator[](int j) const { return bf16_bits_to_f32(a[j]); }
  GFA_DEV void load(const bf16* p) { a = *reinterpret_cast<const Vec*>(p); }
  GFA_DEV void load(const bf16* p, int left) {
    const u16* q = reinterpret_cast<const u16*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = j < left ? q[j] : (u16)0;
  }
};
template <typename T>
GFA_DEV void load8(float* v, const T* p, int left) {
  Eight<T> e;
  if (left >= 8)
    e.load(p);
  else
    e.load(p, left);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = e[j];
}
GFA_DEV void store8(float* p, const float* v, int left) {
  using H = typename Eight<float>::Half;
  if (left >= 8) {
    *reinterpret_cast<H*>(p) = H{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<H*>(p + 4) = H{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = v[j];
  }
}
GFA_DEV void store8(bf16* p, const float* v, int left) {
  using V = typename Eight<bf16>::Vec;
  if (left >= 8) {
    V a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = round_raw<bf16>(v[j]);
    *reinterpret_cast<V*>(p) = a;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) put(p + j, v[j]);
  }
}

// v becomes the first of split's two numbers, rest the second
GFA_DEV void split8(float (&v)[8], float (&rest)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    u16 high;
    split(v[j], high, rest[j]);
    v[j] = raw_to_f32(high);
  }
}

// waits until at most N of the wave's pieces are under way and its LDS reads
// are done, then for the block's other waves
template <int N>
GFA_DEV void wait_pieces() {
  static_assert(N < 64, "six bits of vmcnt");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N)
               : "memory");
}

// waits for the block's waves to be done with LDS
GFA_DEV void wait_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

GFA_DEV auto buffer_at(const void* p, long bytes) {
  const long most = 0x7ffffff0;
  return __builtin_amdgcn_make_buffer_rsrc(
      const_cast<void*>(p), 0, (int)max(0l, min(bytes, most)),
      0x00020000);
}

// One operand's way into LDS: pieces of 1 KB, DEPTH k-tiles a stage, shared
// out over the block's waves.
template <typename T, int BX, bool COLS, int WAVES, int DEPTH>
struct Loader {
  using O = Operand<T, BX, COLS>;
  static constexpr int ES = sizeof(T), BK = O::BK;
  static constexpr int kTile = BX / 8;  // pieces of a k-tile
  static constexpr int kPieces = kTile / WAVES * DEPTH;  // a wave's of a stage
  static_assert(kTile % WAVES == 0, "whole pieces a wave");
  static constexpr int kEach = kTile / WAVES;  // a wave's of a k-tile
  const char* at;  // the corner of the next k-tile
  long bytes;      // from there to the operand's end, whose rows end with a
                   // whole granule; of columns, rows behind the last k lie
                   // outside, since none begins before the last one's end
  long step;       // from one k-tile to the next
  int left;        // k from there on
  int wave, lane;
  int offset[kEach];

  // x0: first row (column) of the tile, X: all of them; kb, kn: part of k
  Loader() = default;
  GFA_DEV Loader(const T* p, long stride, long x0, long X, long kb, int kn,
                 int wave_, int lane_)
      : left(kn), wave(wave_), lane(lane_) {
    auto whole16 = [](long v) { return (v * ES + 15) & ~15l; };
    at = reinterpret_cast<const char*>(COLS ? p + kb * stride + x0
                                            : p + x0 * stride + kb);
    bytes = COLS ? (kn - 1) * stride * ES + whole16(X) - x0 * ES
                 : (X - x0 - 1) * stride * ES + whole16(kn);
    step = (COLS ? BK * stride : BK) * ES;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      offset[i] = O::source((i * WAVES + wave) * 64 + lane, (int)stride);
  }

  // back over so many k-tiles, in an operand of the same shape `apart` bytes
  // from this one
  GFA_DEV void rewind(int ktiles, long apart) {
    at += apart - ktiles * step;
    bytes += ktiles * step;
    left += ktiles * BK;
  }

  // A piece of the next k-tile, the i-th of this wave. Past the end nothing is
  // read and zeros arrive, so the counts of pieces under way stay what the
  // waits expect.
  GFA_DEV void piece(char* lds, int i) const {
    int off = offset[i];
    if constexpr (!COLS) {
      // rows: the last k-tile is cut off at the end of k
      const int idx = (i * WAVES + wave) * 64 + lane;
      const int k = ((idx & 7) ^ O::swizzle(idx >> 3)) * (16 / ES);
      if (left < BK && k >= left) off = 0x7ffffff8;
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        buffer_at(at, bytes), (LdsPtr)(lds + (i * WAVES + wave) * 1024), 16,
        off, 0, 0, 0);
  }
  GFA_DEV void advance() {
    at += step;
    bytes -= step;
    left -= BK;
  }

  // the next DEPTH k-tiles
  GFA_DEV void fetch(char* lds) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) piece(lds + d * kTile * 1024, i);
      advance();
    }
  }
};

// One step's instructions in the order that linear_tile wants: for each row of
// fragments its products, then the LDS reads for the next step and its share
// of the PIECES fetched.
template <int FM, int FN, int MFMAS, int READS_A, int READS_B, int PIECES,
          int... I>
GFA_DEV void order(std::integer_sequence<int, I...>) {
  constexpr int kMfma = 0x8, kVmemRead = 0x20, kLdsRead = 0x100;
  ((__builtin_amdgcn_sched_group_barrier(kMfma, FN * MFMAS, 0),
    __builtin_amdgcn_sched_group_barrier(
        kLdsRead,
        ((I + 1) * FN / FM - I * FN / FM) * READS_B + READS_A, 0),
    __builtin_amdgcn_sched_group_barrier(kVmemRead, PIECES / FM, 0)),
   ...);
}

constexpr int kEpilogueRows = 32;
// Block's results, that of work m0, n0 (row mt of tiles) and part
template <typename T, int BM, int BN, int WM, int WN, int EPI>
GFA_DEV void tile_epilogue(const f32x4 (&acc)[BM / WM / 16][BN / WN / 16],
                           char* lds, int wave, int lane, int mt, long n0,
                           int part, const GemmArgs& g,
                           const EpilogueArgs<T>& e, T* c) {
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, FN = TN / 16;
  const long m0 = (long)mt * BM;
  const int wm = wave / WN * TM, wn = wave % WN * TN;
  // Each wave passes ROWS rows at a time through LDS of its own, from the
  // matrix cores' layout to eight neighbouring n a lane: full lines to and
  // from memory, and a loop for the activation, whose code unrolled over all
  // accumulators would not stay in the instruction cache.
  constexpr int ROWS = kEpilogueRows, EROW = TN * 4 + 16;
  constexpr int LPR = TN / 8, RPI = 64 / LPR, ITER = ROWS / RPI;
  char* mine = lds + wave * ROWS * EROW;
  const long n = n0 + wn + (lane % LPR) * 8;
  const int left = (int)max(0l, min(8l, g.N - n));
  const bool whole = n0 + wn + TN <= g.N;
  const bool curved =
      EPI == kSlope || e.act.act != kLinear || e.act.clamp < INFINITY;
  float bias[8] = {};
  if (EPI != kPlain && EPI != kPartial && e.bias && left) {
    if (e.bias_f32)
      load8(bias, static_cast<const float*>(e.bias) + n, left);
    else
      load8(bias, static_cast<const T*>(e.bias) + n, left);
#pragma unroll
    for (int j = 0; j < 8; ++j) bias[j] *= e.bias_gain;
  }
  const T* op = EPI == kForward ? e.residual : EPI == kSlope ? e.dy : nullptr;
  const long os = EPI == kForward ? e.res_stride : e.dy_stride;
  float sums[8] = {};
#pragma unroll
  for (int h = 0; h < TM / ROWS; ++h) {
    const long mh = m0 + wm + h * ROWS + lane / LPR;
    char* at = mine + lane / LPR * EROW + (lane % LPR) * 32;
    // Residual or dy: all asked for before the first store, which would hold
    // up what waits for a load behind it. Rows past the last repeat it.
    Eight<T> other[ITER];
    if (op && whole) {
#pragma unroll
      for (int q = 0; q < ITER; ++q)
        other[q].load(op + min(mh + q * RPI, g.M - 1) * os + n);
    } else if (op) {
#pragma unroll
      for (int q = 0; q < ITER; ++q)
        other[q].load(op + min(mh + q * RPI, g.M - 1) * os + n, left);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        *reinterpret_cast<f32x4*>(mine + (i * 16 + (lane & 15)) * EROW +
                                  (j * 16 + (lane >> 4) * 4) * 4) =
            acc[h * (ROWS / 16) + i][j];
    __builtin_amdgcn_wave_barrier();
    auto read = [&](float (&z)[8], int q) {
      const f32x4* p = reinterpret_cast<const f32x4*>(at + q * RPI * EROW);
      const f32x4 v[2] = {p[0], p[1]};
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = v[j / 4][j % 4];
    };
    if ((EPI == kForward || EPI == kSlope) && curved) {
      // the activation, stored at once or back to meet the operands
#pragma unroll 1
      for (int q = 0; q < ITER; ++q) {
        const long m = mh + q * RPI;
        float z[8];
        read(z, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = g.alpha * z[j] + bias[j];
        if (EPI == kForward && e.z && m < g.M)
          store8(e.z + m * g.N + n, z, left);
        if (EPI == kForward)
          act_values(z, e.act);
        else
          act_slopes(z, e.act);
        if (op) {
          f32x4* p = reinterpret_cast<f32x4*>(at + q * RPI * EROW);
          p[0] = f32x4{z[0], z[1], z[2], z[3]};
          p[1] = f32x4{z[4], z[5], z[6], z[7]};
        } else if (m < g.M) {
          store8(c + m * g.ldc + n, z, left);
        }
      }
      if (!op) continue;
    }
#pragma unroll
    for (int q = 0; q < ITER; ++q) {
      const long m = mh + q * RPI;
      float z[8];
      read(z, q);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (EPI == kPlain) z[j] *= g.alpha;
        if (EPI == kForward && !curved)
          z[j] = e.act.gain * (g.alpha * z[j] + bias[j]);
        if (EPI == kForward && op) z[j] += other[q][j];
        if (EPI == kSlope) z[j] *= other[q][j];
      }
      // 0 behind the last column, where an infinite x makes z no number
      if (EPI == kSlope && !whole)
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = j < left ? z[j] : 0.f;
      if (m >= g.M) continue;
      if constexpr (EPI == kSlope) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[j] += z[j];
        // dz has padded rows, zero behind the last element
        if (left) {
          if constexpr (sizeof(T) == 2) {
            float rest[8];
            split8(z, rest);
            store8(e.dz_low + m * g.ldc + n, rest, 8);
          }
          store8(c + m * g.ldc + n, z, 8);
        }
      } else if constexpr (EPI == kPartial) {
        store8(e.partial + (part * g.M + m) * g.N + n, z, left);
      } else {
        store8(c + m * g.ldc + n, z, left);
      }
    }
  }
  if (EPI == kSlope && e.partial) {
    // the block's sums over its rows: lanes of the same columns, then the
    // waves one above the other
#pragma unroll
    for (int j = 0; j < 8; ++j)
      for (int o = LPR; o < 64; o <<= 1) sums[j] += __shfl_xor(sums[j], o);
    __syncthreads();
    float* s = reinterpret_cast<float*>(lds);
    if (lane < LPR)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s[wave / WN * BN + wn + lane * 8 + j] = sums[j];
    __syncthreads();
    for (int i = threadIdx.x; i < BN; i += WAVES * 64) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WM; ++w) v += s[w * BN + i];
      if (n0 + i < g.N) e.partial[(long)mt * g.N + n0 + i] = v;
    }
  }
}

template <typename T, int BM, int BN, int WM, int WN, bool ACOLS, bool BCOLS,
          int EPI>
__global__ __launch_bounds__(WM * WN * 64)
void linear_tile(GemmArgs g, EpilogueArgs<T> e, T* __restrict__ c,
                 const T* __restrict__ a, const T* __restrict__ b) {
  using OA = Operand<T, BM, ACOLS>;
  using OB = Operand<T, BN, BCOLS>;
  using F = Frag<T>;
  constexpr int BK = OA::BK, WAVES = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int kStage = OA::kBytes + OB::kBytes;
  constexpr int kEpi = WAVES * kEpilogueRows * (TN * 4 + 16);
  // Tiles of 256 in bf16: a block takes one after the other, and the next
  // one's first pieces come in during the epilogue (65536x512x2048: 185 us,
  // 199 us with a block a tile). Products of floats take five times as long,
  // and what the next tile needs would not stay in registers beside them.
  constexpr bool AHEAD = BM == 256 && sizeof(T) == 2;
  constexpr int kEpiAt = AHEAD ? kStage : 0;
  constexpr int kLds =
      2 * kStage > kEpiAt + kEpi ? 2 * kStage : kEpiAt + kEpi;
  __shared__ __attribute__((aligned(16))) char lds[kLds];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // Work: an XCD's blocks (every eighth) take neighbouring tiles of one part
  // of k, in groups of 4 rows of tiles, so that they share operands in its
  // L2 (all tiles of a part, where there are few).
  const int tm = (int)((g.M + BM - 1) / BM), tn = (int)((g.N + BN - 1) / BN);
  const int parts = (int)((g.K + g.k_split - 1) / g.k_split);
  const int total = tm * tn * parts, per = (total + 7) / 8;
  const int end = min(total, ((int)(blockIdx.x & 7) + 1) * per);
  int work = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (work >= end) return;
  int part, mt;
  long n0;
  using LA = Loader<T, BM, ACOLS, WAVES, 1>;
  using LB = Loader<T, BN, BCOLS, WAVES, 1>;
  LA load_a;
  LB load_b;
  // dx and dw of bf16: the product goes over k again with the rest of dz
  constexpr bool TWICE = BCOLS && sizeof(T) == 2;
  bool again = false;
  auto place = [&] {
    part = work / (tm * tn);
    const int tile = work - part * tm * tn;
    const int group = tile / (4 * tn), in_group = tile - group * 4 * tn;
    const int rows = min(4, tm - group * 4);
    mt = group * 4 + in_group % rows;
    n0 = (long)(in_group / rows) * BN;
    const long kb = part * g.k_split;
    const int kn = (int)min(g.K - kb, g.k_split);
    load_a = LA(a, g.lda, (long)mt * BM, g.M, kb, kn, wave, lane);
    load_b = LB(b, g.ldb, n0, g.N, kb, kn, wave, lane);
    if (TWICE) again = e.a_low;
    return (kn + BK - 1) / BK * (again ? 2 : 1);
  };
  int tiles = place();
  constexpr int kPieces = LA::kPieces + LB::kPieces;
  auto piece = [&](char* to, int p) {
    if (p < LA::kEach)
      load_a.piece(to, p);
    else
      load_b.piece(to + OA::kBytes, p - LA::kEach);
  };
  auto advance = [&] {
    load_a.advance();
    load_b.advance();
    if (TWICE && again && load_a.left <= 0) {
      load_a.rewind(tiles / 2, (e.a_low - a) * (long)sizeof(T));
      load_b.rewind(tiles / 2, 0);
      again = false;
    }
  };
  // the next k-tile
  auto fetch = [&](char* to) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) piece(to, p);
    advance();
  };

  const int wm = wave / WN * TM, wn = wave % WN * TN;
  f32x4 acc[FM][FN];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{};
  };
  // n along the rows of the result, so that a lane holds four neighbours:
  // b is the left operand.
  struct Frags {
    typename F::Type a[FM], b[FN];
  };
  auto read_a = [&](Frags& f, const char* from, int step, int i) {
    f.a[i] = F::template read<BM, ACOLS>(from, wm + i * 16, step, lane);
  };
  auto read_b = [&](Frags& f, const char* from, int step, int j) {
    f.b[j] = F::template read<BN, BCOLS>(from + OA::kBytes, wn + j * 16, step,
                                         lane);
  };
  if constexpr (BM == 256) {
    // One block a CU: while one of a k-tile's two steps is multiplied, the
    // fragments of the next are read, a row's as soon as the row before it is
    // done with, and the k-tile after next is fetched into the half that was
    // read last (8192x4096x4096 bf16: 234 us, 263 us as below).
    Frags f0, f1;
    // next: the step's fragments in `from`; pieces go to `to`
    auto multiply = [&](const Frags& f, Frags& next, const char* from,
                        int step, char* to, auto pieces) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = F::mma(f.b[j], f.a[i], acc[i][j]);
#pragma unroll
        for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j)
          read_b(next, from, step, j);
        read_a(next, from, step, i);
        if (pieces())
#pragma unroll
          for (int p = i * kPieces / FM; p < (i + 1) * kPieces / FM; ++p)
            piece(to, p);
      }
      order<FM, FN, F::kMfmas, ACOLS ? F::kColReads : 1,
            BCOLS ? F::kColReads : 1, pieces()>(
          std::make_integer_sequence<int, FM>{});
    };
    // A k-tile's second step and the next one's first. Where the compiler
    // cannot tell that no piece goes to where fragments are read, it lets
    // transposed reads wait for all pieces under way (8192x4096x4096 bf16: dx
    // 235 us, 267 us so; dw 216 us, 245 us so).
    auto both = [&](const char* __restrict__ from, char* __restrict__ to) {
      multiply(f1, f0, from, 0, to, std::integral_constant<int, kPieces>{});
      multiply(f0, f1, from, 1, nullptr, std::integral_constant<int, 0>{});
      advance();
    };
    fetch(lds);
    for (;;) {
      clear();
      fetch(lds + kStage);
      wait_pieces<kPieces>();
#pragma unroll
      for (int j = 0; j < FN; ++j) read_b(f0, lds, 0, j);
#pragma unroll
      for (int i = 0; i < FM; ++i) read_a(f0, lds, 0, i);
      multiply(f0, f1, lds, 1, nullptr, std::integral_constant<int, 0>{});
      for (int t = 1; t < tiles; ++t) {
        wait_pieces<0>();
        both(lds + (t & 1) * kStage, lds + (~t & 1) * kStage);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = F::mma(f1.b[j], f1.a[i], acc[i][j]);
      wait_pieces<0>();  // the epilogue writes where the pieces go
      const int row = mt, p = part;
      const long col = n0;
      work = AHEAD ? work + gridDim.x / 8 : end;
      if (work < end) {
        tiles = place();
        fetch(lds);
      }
      tile_epilogue<T, BM, BN, WM, WN, EPI>(acc, lds + kEpiAt, wave, lane,
                                            row, col, p, g, e, c);
      if (work >= end) return;
      wait_lds();
    }
  } else {
    // Several blocks a CU fill each other's gaps, and a simple order leaves
    // them the registers (524288x128x128 bf16: dx 52 us, 56 us as above).
    auto multiply = [&](const char* __restrict__ from, char* __restrict__ to,
                        bool more) {
      if (more) fetch(to);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Frags f;
#pragma unroll
        for (int j = 0; j < FN; ++j) read_b(f, from, s, j);
#pragma unroll
        for (int i = 0; i < FM; ++i) read_a(f, from, s, i);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[i][j] = F::mma(f.b[j], f.a[i], acc[i][j]);
      }
    };
    clear();
    fetch(lds);
    for (int t = 0; t < tiles; ++t) {
      wait_pieces<0>();
      multiply(lds + (t & 1) * kStage, lds + (~t & 1) * kStage,
               t + 1 < tiles);
    }
    wait_pieces<0>();  // the epilogue writes where the pieces go
    tile_epilogue<T, BM, BN, WM, WN, EPI>(acc, lds + kEpiAt, wave, lane, mt,
                                          n0, part, g, e, c);
  }
}

// The epilogue of four neighbouring sums of row m, from column n on. What it
// reads besides can be asked for before the sums are there.
template <typename T, int EPI>
struct Finish4 {
  long m, n;
  int left;  // how many of the four lie within the matrix
  float bias[4];
  typename Raw<T>::type other[4];

  GFA_DEV Finish4(long m_, long n_, const GemmArgs& g,
                  const EpilogueArgs<T>& e)
      : m(m_), n(n_), left(m_ < g.M ? (int)max(0l, min(4l, g.N - n_)) : 0) {
    if constexpr (EPI == kForward || EPI == kSlope) {
      const T* p = EPI == kForward ? e.residual : e.dy;
      if (p) p += m * (EPI == kForward ? e.res_stride : e.dy_stride) + n;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bias[j] = 0.f;
        other[j] = 0;
        if (j < left) {
          if (e.bias)
            bias[j] = e.bias_gain *
                      (e.bias_f32
                           ? static_cast<const float*>(e.bias)[n + j]
                           : to_f32(static_cast<const T*>(e.bias)[n + j]));
          if (p)
            other[j] = reinterpret_cast<const typename Raw<T>::type*>(p)[j];
        }
      }
    }
  }

  // the sums become what was written, 0 outside the matrix
  GFA_DEV void write(float (&o)[4], const GemmArgs& g,
                     const EpilogueArgs<T>& e, T* c) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= g.alpha;
    if constexpr (EPI == kForward || EPI == kSlope) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += bias[j];
      if (EPI == kForward && e.z)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) e.z[m * g.N + n + j] = o[j];
      if (EPI == kForward)
        act_values(o, e.act);
      else
        act_slopes(o, e.act);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float r = raw_to_f32(other[j]);
        o[j] = EPI == kForward ? o[j] + r : o[j] * r;
      }
    }
    // dz has rows padded to eight, zero behind the last element
    const int end = EPI == kSlope ? (m < g.M ? (int)(g.ldc - n) : 0) : left;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= left) o[j] = 0.f;
      if (j < end) {
        auto raw = round_raw<T>(o[j]);
        if constexpr (EPI == kSlope && sizeof(T) == 2) {
          float rest;
          split(o[j], raw, rest);
          put(e.dz_low + m * g.ldc + n + j, rest);
        }
        *reinterpret_cast<typename Raw<T>::type*>(c + m * g.ldc + n + j) = raw;
      }
    }
  }
};

// The sums of a block's four waves over 16 FM x 16 FN of C meet in LDS and
// go through the epilogue, four neighbouring n of one m a thread.
template <typename T, int EPI, int FM, int FN>
GFA_DEV void join_waves(const f32x4 (&acc)[FM][FN], char* lds, long n0, int mt,
                        const Finish4<T, EPI>& finish, const GemmArgs& g,
                        const EpilogueArgs<T>& e, T* c) {
  constexpr int BM = 16 * FM, BN = 16 * FN, WAVES = 4;
  constexpr int ROW = BN * 4 + 16;  // bytes
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<f32x4*>(lds + (wave * BM + i * 16 + (lane & 15)) * ROW +
                                (j * 16 + (lane >> 4) * 4) * 4) = acc[i][j];
  __syncthreads();
  const int row = threadIdx.x / (BN / 4), col = threadIdx.x % (BN / 4) * 4;
  float o[4] = {};
  if (row < BM) {
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      v += *reinterpret_cast<f32x4*>(lds + (w * BM + row) * ROW + col * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = v[j];
    if constexpr (EPI == kPartial) {
      float* p =
          e.partial + ((long)blockIdx.y * g.M + finish.m) * g.N + finish.n;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < finish.left) p[j] = o[j];
    } else {
      finish.write(o, g, e, c);
    }
  }
  if (EPI == kSlope && e.partial) {
    __syncthreads();
    if (row < BM)
      *reinterpret_cast<f32x4*>(lds + row * ROW + col * 4) =
          f32x4{o[0], o[1], o[2], o[3]};
    __syncthreads();
    if (threadIdx.x < BN && n0 + threadIdx.x < g.N) {
      float s = 0.f;
      for (int r = 0; r < BM; ++r)
        s += *reinterpret_cast<float*>(lds + r * ROW + threadIdx.x * 4);
      e.partial[(long)mt * g.N + n0 + threadIdx.x] = s;
    }
  }
}

// the part of C that join_waves gives a thread
template <typename T, int EPI, int FM, int FN>
GFA_DEV Finish4<T, EPI> thread_part(long m0, long n0, const GemmArgs& g,
                                    const EpilogueArgs<T>& e) {
  const int row = threadIdx.x / (FN * 4);
  return {row < FM * 16 ? m0 + row : g.M, n0 + threadIdx.x % (FN * 4) * 4, g,
          e};
}

// eight bf16 or four floats of a row at any alignment, as a fragment
template <typename T>
GFA_DEV typename Frag<T>::Type load16(const T* p) {
  return *reinterpret_cast<const typename Unaligned<T>::Vec*>(p);
}
template <typename T>
GFA_DEV typename Frag<T>::Type load16(const T* p, int left) {
  typename Frag<T>::Type v{};
#pragma unroll
  for (int j = 0; j < 16 / (int)sizeof(T); ++j)
    if (j < left) v[j] = reinterpret_cast<const typename Raw<T>::type*>(p)[j];
  return v;
}

// Products with at most 32 rows (rows times rows only): 16 FM x 16 of C a
// block, so that the weights, each read once, come in over as many CUs as
// there are; k is shared out over the block's four waves in chunks of 256
// bytes. Fragments come straight from memory, two chunks a wave under way,
// with no barrier before the waves meet; a row needs no alignment. Latency
// bounds it: 1x1024x4096 bf16 takes 4.1 us (8.4 MB, 1.6 us at a copy's rate)
// and 17x512x512 float 5.5 us, where tiles of 32x32 by way of LDS took 7.3
// and 7.2 us, and an empty launch in a graph 1.5 us.
template <typename T, int FM, int EPI>
__global__ __launch_bounds__(256)
void linear_direct(GemmArgs g, EpilogueArgs<T> e, T* __restrict__ c,
                   const T* __restrict__ a, const T* __restrict__ b) {
  constexpr int FN = 1, WAVES = 4, U = 4;
  using F = Frag<T>;
  constexpr int STEP = F::kStep, V = 16 / sizeof(T);
  __shared__
      __attribute__((aligned(16))) char lds[WAVES * FM * 16 * (64 + 16)];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long n0 = (long)blockIdx.x * 16;
  const long kb = (long)blockIdx.y * g.k_split;
  const int kn = (int)min(g.K - kb, g.k_split);
  const auto finish = thread_part<T, EPI, FM, FN>(0, n0, g, e);

  // rows past the last repeat it; their sums are not stored
  const int lane_k = (lane >> 4) * V;
  const T* pa[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i)
    pa[i] = a + min(i * 16l + (lane & 15), g.M - 1) * g.lda + kb + lane_k;
  const T* pb = b + min(n0 + (lane & 15), g.N - 1) * g.ldb + kb + lane_k;
  f32x4 acc[FM][FN] = {};
  struct Chunk {
    typename F::Type a[U][FM], b[U];
  };
  auto load = [&](Chunk& q, int chunk) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (chunk * U + u) * STEP;
      q.b[u] = load16<T>(pb + k);
#pragma unroll
      for (int i = 0; i < FM; ++i) q.a[u][i] = load16<T>(pa[i] + k);
    }
  };
  auto mma = [&](const Chunk& q) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < FM; ++i)
        acc[i][0] = F::mma(q.b[u], q.a[u][i], acc[i][0]);
  };
  const int chunks = kn / (U * STEP);
  Chunk q0, q1;
  if (wave < chunks) load(q0, wave);
  for (int q = wave; q < chunks; q += 2 * WAVES) {
    const bool more = q + WAVES < chunks;
    if (more) load(q1, q + WAVES);
    mma(q0);
    if (!more) break;
    if (q + 2 * WAVES < chunks) load(q0, q + 2 * WAVES);
    mma(q1);
  }
  // what is left of k, a step a wave, the last one cut off
  for (int k = (chunks * U + wave) * STEP; k < kn; k += WAVES * STEP) {
    const int left = kn - k - lane_k;
    const auto fb = load16<T>(pb + k, left);
#pragma unroll
    for (int i = 0; i < FM; ++i)
      acc[i][0] = F::mma(fb, load16<T>(pa[i] + k, left), acc[i][0]);
  }
  join_waves<T, EPI, FM, FN>(acc, lds, n0, 0, finish, g, e, c);
}

// Products that tiles of 64x64 spread over too few CUs: 32x32 of C a block.
// The four waves share out k instead of C (each takes every fourth step of
// all 32x32), so a block's operands pass through LDS once and its time falls
// with k alone; their sums meet in LDS. Where that still leaves CUs idle, k
// is split over blocks too (kPartial). 544x512x512: 5.8 us bf16, 10.2 us
// float (tiles of 64: 6.7 and 14.8 us). The product itself is 1.9 us of the
// whole card's float rate; 272 blocks put two on some of the 256 CUs, which is
// 3.4 us there, and the rest is the latency of eight short stages one after
// the other and of the launch.
constexpr int kSmallLds = 4 * 2 * 2 * 32 * 128;  // stages, operands, depth
template <typename T, bool ACOLS, bool BCOLS, int EPI>
GFA_DEV void small_block(char* lds, int block, const GemmArgs& g,
                         const EpilogueArgs<T>& e, T* c, const T* a,
                         const T* b, const T* a_low = nullptr) {
  constexpr int B = 32, DEPTH = 2, STAGES = 4, WAVES = 4, FM = 2, FN = 2;
  using OA = Operand<T, B, ACOLS>;
  using F = Frag<T>;
  constexpr int kHalf = OA::kBytes * DEPTH, kStage = 2 * kHalf;
  static_assert(STAGES * kStage == kSmallLds, "what the callers give");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tn = (int)((g.N + B - 1) / B);
  const int mt = block / tn;
  const long m0 = (long)mt * B, n0 = (long)(block % tn) * B;
  const long kb = (long)blockIdx.y * g.k_split;
  const int kn = (int)min(g.K - kb, g.k_split);
  const auto finish = thread_part<T, EPI, FM, FN>(m0, n0, g, e);

  using LA = Loader<T, B, ACOLS, WAVES, DEPTH>;
  using LB = Loader<T, B, BCOLS, WAVES, DEPTH>;
  f32x4 acc[2][2] = {};
  const int tiles = (kn + DEPTH * OA::BK - 1) / (DEPTH * OA::BK);
  // a k-tile holds two steps, a stage four: one for each wave
  const int tile_of = wave / 2 * OA::kBytes, step = wave % 2;
  for (const T* left = a; left; left = left == a ? a_low : nullptr) {
    LA load_a(left, g.lda, m0, g.M, kb, kn, wave, lane);
    LB load_b(b, g.ldb, n0, g.N, kb, kn, wave, lane);
    auto fetch = [&](int stage) {
      load_a.fetch(lds + stage * kStage);
      load_b.fetch(lds + stage * kStage + kHalf);
    };
    auto multiply = [&](const char* __restrict__ from, char* __restrict__ to) {
      load_a.fetch(to);
      load_b.fetch(to + kHalf);
      const char* pa = from + tile_of;
      const char* pb = pa + kHalf;
      typename F::Type fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = F::template read<B, ACOLS>(pa, i * 16, step, lane);
        fb[i] = F::template read<B, BCOLS>(pb, i * 16, step, lane);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = F::mma(fb[j], fa[i], acc[i][j]);
    };
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) fetch(t);
    for (int t = 0; t < tiles; ++t) {
      wait_pieces<(STAGES - 2) * (LA::kPieces + LB::kPieces)>();
      multiply(lds + t % STAGES * kStage,
               lds + (t + STAGES - 1) % STAGES * kStage);
    }
    wait_pieces<0>();  // the next operand, or the sums, go where pieces went
  }
  join_waves<T, EPI, FM, FN>(acc, lds, n0, mt, finish, g, e, c);
}

template <typename T, bool ACOLS, bool BCOLS, int EPI>
__global__ __launch_bounds__(256)
void linear_small(GemmArgs g, EpilogueArgs<T> e, T* __restrict__ c,
                  const T* __restrict__ a, const T* __restrict__ b) {
  __shared__ __attribute__((aligned(16))) char lds[kSmallLds];
  small_block<T, ACOLS, BCOLS, EPI>(
      lds, blockIdx.x, g, e, c, a, b,
      BCOLS && sizeof(T) == 2 ? e.a_low : nullptr);
}

// out[i] = scale * sum_r src[r][i] for eight columns from n0 on
template <typename S>
GFA_DEV void sum_columns(char* lds, const S* src, long stride, long rows,
                         int n, int n0, float scale, void* out, bool out_f32) {
  const int c = threadIdx.x & 7, q = threadIdx.x >> 3, i = n0 + c;
  float* red = reinterpret_cast<float*>(lds);
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (long r = q; r < rows; r += 32) s += to_f32(src[r * stride + i]);
  }
  red[c * 33 + q] = s;
  __syncthreads();
  if (threadIdx.x < 8 && i < n) {
    s = 0.f;
    for (int k = 0; k < 32; ++k) s += red[c * 33 + k];
    s *= scale;
    if (out_f32)
      static_cast<float*>(out)[i] = s;
    else
      put(static_cast<bf16*>(out) + i, s);
  }
}

// A small layer's whole backward after dz: blocks of dw, of dx and of db
// side by side. One launch for three costs the host less, and neither
// product alone fills the card.
template <typename T>
__global__ __launch_bounds__(256)
void linear_backward_small(SmallBackward<T> p) {
  __shared__ __attribute__((aligned(16))) char lds[kSmallLds];
  const EpilogueArgs<T> none{};
  int block = blockIdx.x;
  if (block < p.dw_blocks) {
    small_block<T, true, true, kPlain>(lds, block, p.dw, none, p.dw_out, p.dz,
                                       p.x, p.dz_low);
    return;
  }
  block -= p.dw_blocks;
  if (block < p.dx_blocks) {
    small_block<T, false, true, kPlain>(lds, block, p.dx, none, p.dx_out, p.dz,
                                        p.w, p.dz_low);
    return;
  }
  block -= p.dx_blocks;
  if (p.partial)
    sum_columns(lds, p.partial, p.n, p.groups, p.n, block * 8, p.db_scale,
                p.db_out, p.db_f32);
  else
    sum_columns(lds, p.dz, p.dw.lda, p.dw.K, p.n, block * 8, p.db_scale,
                p.db_out, p.db_f32);
}

// The epilogue over sums of k split over blocks; four n a thread.
template <typename T, int EPI>
__global__ __launch_bounds__(256)
void linear_finish(GemmArgs g, EpilogueArgs<T> e, T* __restrict__ c,
                   int splits) {
  const long wide = (g.N + 3) / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long m = i / wide, n = i % wide * 4;
  if (m >= g.M) return;
  const Finish4<T, EPI> finish(m, n, g, e);
  const float* p = e.partial + m * g.N + n;
  float o[4] = {};
#pragma unroll 8
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] += j < finish.left ? p[s * g.M * g.N + j] : 0.f;
  finish.write(o, g, e, c);
}

// C = alpha * sum of the parts of k: eight elements a thread, the threads of
// a block side by side or, for many parts, `groups` of them one above the
// other, each for every so manieth part.
template <typename T>
__global__ __launch_bounds__(256)
void sum_splits(T* __restrict__ c, const float* __restrict__ partial,
                int splits, long count, float alpha, int groups) {
  __shared__ __attribute__((aligned(16))) float red[256 * 8];
  const int wide = 256 / groups;
  const int col = threadIdx.x % wide, q = threadIdx.x / wide;
  const long i = ((long)blockIdx.x * wide + col) * 8;
  const int left = (int)max(0l, min(8l, count - i));
  float s[8] = {};
  if (left == 8) {
#pragma unroll 4
    for (int k = q; k < splits; k += groups) {
      Eight<float> v;
      v.load(partial + k * count + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
  } else if (left) {
    for (int k = q; k < splits; k += groups)
      for (int j = 0; j < 8; ++j)
        if (j < left) s[j] += partial[k * count + i + j];
  }
  if (groups > 1) {
    f32x4* mine = reinterpret_cast<f32x4*>(red + threadIdx.x * 8);
    mine[0] = f32x4{s[0], s[1], s[2], s[3]};
    mine[1] = f32x4{s[4], s[5], s[6], s[7]};
    __syncthreads();
    if (q) return;
    for (int g = 1; g < groups; ++g) {
      const f32x4* v =
          reinterpret_cast<const f32x4*>(red + (g * wide + col) * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j / 4][j % 4];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] *= alpha;
  if (left) store8(c + i, s, left);
}

// dst[r][0..width) = src[r][0..n), zero behind: 16-byte rows for the tiles,
// in a pass of their own, which costs less than element loads in every
// block that reads a row (1037x515x771: 3.8 us of 15)
template <typename T>
__global__ __launch_bounds__(256)
void pad_rows(PadArgs<T> p0, PadArgs<T> p1) {
  const PadArgs<T>& p = blockIdx.y ? p1 : p0;
  const int wide = p.width / 8;
  const long count = p.rows * wide;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count;
       i += (long)gridDim.x * 256) {
    const long r = i / wide;
    const int col = (int)(i - r * wide) * 8;
    float v[8];
    load8(v, p.src + r * p.stride + col, min(8, p.n - col));
    store8(p.dst + r * p.width + col, v, 8);
  }
}

// one tensor or two
template <typename T>
void launch_pad_rows(const PadArgs<T>& p0, const PadArgs<T>& p1,
                     hipStream_t s) {
  auto work = [](const PadArgs<T>& p) {
    return p.dst ? (p.rows * (p.width / 8) + 255) / 256 : 0l;
  };
  const long most = work(p0) > work(p1) ? work(p0) : work(p1);
  hipLaunchKernelGGL(pad_rows<T>,
                     dim3((unsigned)(most < 4096 ? most : 4096),
                          p1.dst ? 2 : 1),
                     dim3(256), 0, s, p0, p1);
}

namespace {

// Microseconds that a CU spends on one k-tile of a block, alone on it or with
// others, and on the rest of a block's work. Measured: 8192x4096x4096 bf16
// takes 234, 314 and 439 us with tiles of 256, 128 and 64, 4096^3 float 940,
// 1021 and 1089 us; 524288x128x128 bf16, half of whose tiles of 256 would be
// padding, 120 us with those and 48 us with 128. Fitted to 21 shapes in both
// types, each cut in up to 40 ways, and put right where a choice lost since
// (2048x4096x2048 bf16: 50 us with 128, 53 us with 64).
struct TileCost {
  int side;
  double alone, shared, rest;
};
const TileCost kTileCosts[2][5] = {
    // bf16
    {{256, 1.7, 1.7, 8}, {128, 0.77, 0.57, 2}, {64, 0.40, 0.214, 1},
     {32, 0.2, 0.16, 0.5}, {16, 0.06, 0.05, 0.5}},
    // float
    {{256, 7.4, 7.4, 8}, {128, 2.15, 2.0, 2}, {64, 0.65, 0.53, 1},
     {32, 0.24, 0.21, 0.5}, {16, 0.165, 0.15, 0.5}}};

template <typename T, bool ACOLS, bool BCOLS, int EPI>
void launch_tile(int tile, T* c, const T* a, const T* b, const GemmArgs& g,
                 const EpilogueArgs<T>& e, int splits, hipStream_t s) {
  if constexpr (!ACOLS && !BCOLS) {
    if (tile == 16) {
      const dim3 grid((unsigned)ceil_div(g.N, 16), splits);
      if (g.M <= 16)
        hipLaunchKernelGGL((linear_direct<T, 1, EPI>), grid, dim3(256), 0, s,
                           g, e, c, a, b);
      else
        hipLaunchKernelGGL((linear_direct<T, 2, EPI>), grid, dim3(256), 0, s,
                           g, e, c, a, b);
      return;
    }
  }
  const long tiles = ceil_div(g.M, tile) * (long)ceil_div(g.N, tile);
  // one block a CU for bf16 tiles of 256
  const long blocks = (tiles * splits + 7) / 8 * 8;
  const dim3 grid((unsigned)(tile == 256 && sizeof(T) == 2
                                 ? std::min(blocks, 256l)
                                 : blocks));
#define LAUNCH(B, WM, WN)                                                     \
  hipLaunchKernelGGL((linear_tile<T, B, B, WM, WN, ACOLS, BCOLS, EPI>),       \
                     grid, dim3(WM * WN * 64), 0, s, g, e, c, a, b)
  if (tile == 256)
    LAUNCH(256, 2, 4);
  else if (tile == 128)
    LAUNCH(128, 2, 2);
  else if (tile == 64)
    LAUNCH(64, 2, 2);
  else
    hipLaunchKernelGGL((linear_small<T, ACOLS, BCOLS, EPI>),
                       dim3((unsigned)tiles, splits), dim3(256), 0, s, g, e, c,
                       a, b);
#undef LAUNCH
}

}  // namespace

// linear_direct's rows
bool linear_reads_any_rows(long M) { return M <= 32; }

// The tile and the number of parts of k for which the busiest CU is done
// first: rounds of blocks over 256 CUs, each of so many k-tiles, and for
// parts a launch more that reads their sums again.
LinearPlan linear_plan(long M, long N, long K, bool f32, LinearKind kind) {
  const long ktiles = (K + (f32 ? 31 : 63)) / (f32 ? 32 : 64);
  LinearPlan best{};
  double least = 1e30;
  for (const TileCost& t : kTileCosts[f32]) {
    const bool direct = t.side == 16;
    if (direct != (kind <= kSlopes && linear_reads_any_rows(M))) continue;
    const long blocks =
        direct ? (N + 15) / 16
               : ((M + t.side - 1) / t.side) * ((N + t.side - 1) / t.side);
    // one part, or as many as fill so many rounds, of 8 k-tiles at least
    for (int fill = 0; fill <= 8; ++fill) {
      const long s = fill ? std::min(256 * fill / blocks, ktiles / 8) : 1;
      if (fill && (s < 2 || kind == kSlopes)) continue;
      const long each = (ktiles + s - 1) / s;
      const long rounds = (blocks * s + 255) / 256;
      double cost = rounds == 1 ? each * t.alone + t.rest
                                : rounds * (each * t.shared + t.rest);
      if (s > 1) cost += 3 + 2e-6 * s * M * N;
      if (cost < least) {
        least = cost;
        best = {t.side, (int)s};
      }
    }
  }
  return best;
}

int linear_row_tiles(const LinearPlan& p, long M) {
  return p.tile == 16 ? 1 : ceil_div(M, p.tile);
}

namespace {

// C in one launch, or by splits of k and a launch that sums them
template <typename T, bool ACOLS, bool BCOLS, int EPI>
void launch_split(T* c, const T* a, const T* b, GemmArgs g,
                  EpilogueArgs<T> e, const LinearPlan& p, hipStream_t s) {
  int splits = p.splits;
  if (splits > 1) {
    const long bk = 128 / sizeof(T);
    g.k_split = ((g.K + splits - 1) / splits + bk - 1) / bk * bk;
    splits = (int)((g.K + g.k_split - 1) / g.k_split);
  }
  const int tile = p.tile;
  if (splits == 1) {
    launch_tile<T, ACOLS, BCOLS, EPI>(tile, c, a, b, g, e, 1, s);
    return;
  }
  launch_tile<T, ACOLS, BCOLS, kPartial>(tile, c, a, b, g, e, splits, s);
  if (EPI == kPlain) {
    const long count = g.M * g.N;
    // a thread for every four parts, as long as there are threads to fill
    int groups = 1;
    while (groups < 64 && groups * 4 < splits && count / 8 * groups < 1 << 19)
      groups *= 2;
    hipLaunchKernelGGL(sum_splits<T>,
                       dim3(ceil_div(count, 2048 / groups)), dim3(256), 0, s,
                       c, e.partial, splits, count, g.alpha, groups);
  } else {
    hipLaunchKernelGGL((linear_finish<T, EPI>),
                       dim3(ceil_div(g.M * ((g.N + 3) / 4), 256)), dim3(256),
                       0, s, g, e, c, splits);
  }
}

}  // namespace

template <typename T>
void launch_linear_forward(T* y, const T* x, const T* w, const GemmArgs& g,
                           const EpilogueArgs<T>& e, const LinearPlan& p,
                           hipStream_t s) {
  launch_split<T, false, false, kForward>(y, x, w, g, e, p, s);
}

template <typename T>
void launch_linear_slope(T* dz, const T* x, const T* w, const GemmArgs& g,
                         const EpilogueArgs<T>& e, const LinearPlan& p,
                         hipStream_t s) {
  launch_tile<T, false, false, kSlope>(p.tile, dz, x, w, g, e, 1, s);
}

template <typename T>
void launch_linear_dx(T* dx, float* partial, const T* dz, const T* dz_low,
                      const T* w, const GemmArgs& g, const LinearPlan& p,
                      hipStream_t s) {
  EpilogueArgs<T> e{};
  e.partial = partial;
  e.a_low = dz_low;
  launch_split<T, false, true, kPlain>(dx, dz, w, g, e, p, s);
}

template <typename T>
void launch_linear_dw(T* dw, float* partial, const T* dz, const T* dz_low,
                      const T* x, const GemmArgs& g, const LinearPlan& p,
                      hipStream_t s) {
  EpilogueArgs<T> e{};
  e.partial = partial;
  e.a_low = dz_low;
  launch_split<T, true, true, kPlain>(dw, dz, x, g, e, p, s);
}

// ---- dz from a kept z, and sums over rows ----
// A block takes every so manieth row: `wide` threads of eight columns side
// by side, 256 / wide rows at a time, four of them under way.
template <typename T>
__global__ __launch_bounds__(256)
void linear_dz_kernel(T* __restrict__ dz, T* __restrict__ low,
                      long dz_stride, float* __restrict__ partial,
                      const T* __restrict__ dy,
                      long dy_stride, const float* __restrict__ z,
                      ActParams act, long rows, int n, int wide) {
  constexpr int U = 4;
  __shared__ float red[256][9];
  const int high = 256 / wide, q = threadIdx.x / wide;
  const int i = (blockIdx.x * wide + threadIdx.x % wide) * 8;
  const int left = max(0, min(8, n - i));
  const long step = (long)gridDim.y * high;
  float sum[8] = {};
  for (long r = (long)blockIdx.y * high + q; left && r < rows; r += U * step) {
    Eight<T> d[U];
    Eight<float> zz[U];
    // rows past the last repeat it and are not counted
    if (left == 8) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long at = min(r + u * step, rows - 1);
        d[u].load(dy + at * dy_stride + i);
        if (z) zz[u].load(z + at * n + i);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long at = min(r + u * step, rows - 1);
        d[u].load(dy + at * dy_stride + i, left);
        if (z) zz[u].load(z + at * n + i, left);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * step >= rows) break;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = d[u][j];
      if (z) {
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = zz[u][j];
        act_slopes(s, act);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= s[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += v[j];  // before their rounding
      if (!z) continue;
      // padded rows, zero behind the last element
      const long at = (r + u * step) * dz_stride + i;
      if constexpr (sizeof(T) == 2) {
        float rest[8];
        split8(v, rest);
        store8(low + at, rest, 8);
      }
      store8(dz + at, v, 8);
    }
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[threadIdx.x][j] = sum[j];
  __syncthreads();
  for (int k = threadIdx.x; k < wide * 8; k += 256) {
    const int col = blockIdx.x * wide * 8 + k;
    if (col >= n) break;
    float v = 0.f;
    for (int h = 0; h < high; ++h) v += red[h * wide + k / 8][k % 8];
    partial[(long)blockIdx.y * n + col] = v;
  }
}

namespace {
// threads side by side: as many as a row of n needs, at most a wave's half
int dz_wide(int n) {
  int wide = 1;
  while (wide < 32 && wide * 8 < n) wide *= 2;
  return wide;
}
}  // namespace

// Row groups: at most about two blocks a CU, at least four rows a thread.
int linear_dz_groups(long rows, int n) {
  const int wide = dz_wide(n), high = 256 / wide;
  const long most = (rows + 4 * high - 1) / (4 * high);
  const long want = (512 + ceil_div(n, wide * 8) - 1) / ceil_div(n, wide * 8);
  return (int)(most < want ? most : want);
}

template <typename T>
void launch_linear_dz(T* dz, T* low, long dz_stride, float* partial,
                      const T* dy,
                      long dy_stride, const float* z, const ActParams& act,
                      long rows, int n, hipStream_t s) {
  const int wide = dz_wide(n);
  hipLaunchKernelGGL(linear_dz_kernel<T>,
                     dim3(ceil_div(n, wide * 8), linear_dz_groups(rows, n)),
                     dim3(256), 0, s, dz, low, dz_stride, partial, dy,
                     dy_stride, z, act, rows, n, wide);
}

// One launch where both products' tiles of 32 fit the card a few times over
// and neither k is long (both gradients of 1500x512x512: bf16 14.9 us, float
// 26 us; in launches of their own 18 and 37 us, and two launches more for the
// host). With a dz in two parts, dz included: 544x512x512 bf16 20.5 against
// 24.1 us, 1500x512x512 31.6 against 35.8, near the rule's edge (512x1024x1024)
// 37.5 against 33.6.
bool linear_backward_is_small(long m, long n, long k, bool f32) {
  auto tiles = [](long a, long b) {
    return (long)ceil_div(a, 32) * ceil_div(b, 32);
  };
  return m <= 2048 && n <= 2048 && tiles(m, k) <= 768 && tiles(n, k) <= 1024;
}

template <typename T>
void launch_linear_backward_small(SmallBackward<T> p, hipStream_t s) {
  auto tiles = [](const GemmArgs& g) {
    return ceil_div(g.M, 32) * ceil_div(g.N, 32);
  };
  p.dw_blocks = p.dw_out ? tiles(p.dw) : 0;
  p.dx_blocks = p.dx_out ? tiles(p.dx) : 0;
  const int db_blocks = p.db_out ? ceil_div(p.n, 8) : 0;
  hipLaunchKernelGGL(linear_backward_small<T>,
                     dim3(p.dw_blocks + p.dx_blocks + db_blocks), dim3(256), 0,
                     s, p);
}

#define INSTANTIATE(T)                                                       \
  template void launch_linear_backward_small<T>(SmallBackward<T>,            \
                                                hipStream_t);                \
  template void launch_linear_forward<T>(T*, const T*, const T*,             \
                                         const GemmArgs&,                    \
                                         const EpilogueArgs<T>&,             \
                                         const LinearPlan&, hipStream_t);    \
  template void launch_linear_slope<T>(T*, const T*, const T*,               \
                                       const GemmArgs&,                      \
                                       const EpilogueArgs<T>&,               \
                                       const LinearPlan&, hipStream_t);      \
  template void launch_linear_dx<T>(T*, float*, const T*, const T*,          \
                                    const T*, const GemmArgs&,               \
                                    const LinearPlan&, hipStream_t);         \
  template void launch_linear_dw<T>(T*, float*, const T*, const T*,          \
                                    const T*, const GemmArgs&,               \
                                    const LinearPlan&, hipStream_t);         \
  template void launch_pad_rows<T>(const PadArgs<T>&, const PadArgs<T>&,     \
                                   hipStream_t);                             \
  template void launch_linear_dz<T>(T*, T*, long, float*, const T*, long,    \
                                    const float*, const ActParams&, long,    \
                                    int, hipStream_t);
INSTANTIATE(float)
INSTANTIATE(bf16)

}  // namespace gfa
