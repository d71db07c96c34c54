// Orthogonalised updates: y = x / (|x|_F + eps), then `steps` times g = y y^T, y = a y + (b g + c g g) y,
// and the Muon step that applies the result to a parameter.
//
// The matrices are held with their shorter side (r) as rows (a taller matrix is transposed on the way in and
// out: the polynomial acts on singular values only), padded with zeros to whole tiles.
// Products run on v_mfma_f32_32x32x16_f16 with every fp32 operand x split in two fp16 parts,
//   2^S x = hi + 2^-11 lo,  hi = fp16(2^S x), lo = fp16(2^11 (2^S x - hi)),
// and x y = hi hi' + 2^-11 (hi lo' + lo hi') with fp32 sums of both, on matrix cores that do fp16 at 16 times
// the rate of fp32.  hi is off by at most half a step of 11 bits and lo, which has a sign, by half a step of 11
// more: a pair is within 2^-23 of x, one bit short of fp32, in the same 32 bits; the dropped lo lo' is
// below 2^-22.  lo is as large as hi, so it keeps its bits as far down as hi does: that holds for |2^S x| >= 2^-13,
// and below that a pair is within 2^-36 of 2^S x.  (With lo unscaled its bits were lost below |2^S x| = 2^-2: rows
// 1e-7 of the others were off by 1e-2, now by 5e-6.  The second sum takes registers: 3 % of the time of the
// 128-wide tiles and 2 to 4 % of the small forms.)
// The steps are normalised, so the range is known and the scales are constants: |y| <= 4
// with S = 12 (a head room of 4), |y y^T| <= 16 and |b g + c g g| < 31 with S = 10 (head rooms 4 and 2): y is within
// 2^-23 of its value from 2^-25 on, and within 2^-48 below; g from 2^-23 on, and within 2^-46.
// Against 64 bits the result is as close as the same steps in fp32 where sums are long (the error is theirs,
// not that of the operands), and off by a few 2^-23 a step where one entry makes up a matrix.  Sums are fp32, the
// norm is fp64; the pairs are also where y and g are kept between products: what the products move is what bounds
// them, and an fp32 copy beside the pairs would double it.
//
// A split matrix ("planes") lies in memory as [row][column / 32][part][32]: the two parts of 32 columns are
// one 128-byte line, 8 units of 16 bytes.
//
// Three ways to run the products, by size:
//   both sides <= 128: the whole iteration in one launch, a workgroup per matrix, planes in LDS;
//   few tiles: 32 x 32 tiles (symmetric products: 16 x 16), the contraction split over the waves of a
//     workgroup, operands straight from memory (every load of a wave in flight: a few round trips);
//   otherwise: 64 x 64 or 128 x 128 tiles staged through LDS.
// y y^T and g g are symmetric: only tiles on and below the diagonal are computed, and mirrored.
// Twelve 768 x 2304 (272 GFLOP): 1075 - 1150 us, matrix cores: y y^T 60 us, the polynomial 27, the step of y 113, which is
// 950, 710 and 870 TFLOP/s of fp16 products; norm and first y 50 us each, 5 TB/s.  One 96 x 96: 27 us, 1000 x 257:
// 96 us, the latency of 15 dependent products.
#include "common.h"

#include <algorithm>
#include <cmath>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int PARTS = 64;                  // partial sums of a norm
constexpr float kY = 4096.f, kG = 1024.f;  // 2^S of the planes of y and of g, b g + c g g
constexpr float kLo = 2048.f;              // 2^11: lo parts are held times this
constexpr int ONE = 128;                   // largest side of the one-launch form

struct NsParams {
  // the user's matrices (row-major, as given)
  const float *x;      // Newton-Schulz: input.  Muon: gradient
  float *m, *p, *out;  // Muon: momentum, parameter.  Newton-Schulz: out
  long long ld_x, stride_x, ld_out, stride_out;
  int rows, cols, batch, tall;  // tall: rows > cols
  float momentum, grad_scale, keep, step;
  int nesterov;
  bool flat;  // x (and m) without gaps inside a matrix, 16-byte aligned
  bool vec;   // out / p rows may be written 16 bytes at a time
  float a, b, c, eps;
  int steps;
  // workspace
  int r, n, rp, np;
  _Float16 *yp[2], *gp, *bp;  // planes of y (read and written by one product, so two), g, b g + c g g
  double *sums;               // [batch][PARTS]
};

// ------------------------------------------------------------------------------------- the planes
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split4(f32x4 v, float scale, f16x4 &hi, f16x4 &lo) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 x = {v[2 * h] * scale, v[2 * h + 1] * scale};
    const f16x2 a = __builtin_convertvector(x, f16x2);
    hi[2 * h] = a[0], hi[2 * h + 1] = a[1];
#pragma unroll
    for (int e = 0; e < 2; ++e)  // (one mixed-precision instruction: what is left is exact in fp32)
      lo[2 * h + e] = (_Float16)fmaf((float)a[e], -kLo, v[2 * h + e] * (scale * kLo));
  }
}
// fp16 offset of the hi part of element (row, col) of a matrix of `cols` columns; the lo part lies 32 behind
__device__ __forceinline__ long long plane_at(long long row, int col, int cols) {
  return row * (2ll * cols) + (col >> 5) * 64 + (col & 31);
}
__device__ __forceinline__ void store_split4(_Float16 *at, f32x4 v, float scale) {
  f16x4 hi, lo;
  split4(v, scale, hi, lo);
  *reinterpret_cast<f16x4 *>(at) = hi;
  *reinterpret_cast<f16x4 *>(at + 32) = lo;
}
// Transposed read: lane l of each 16 gets rows 0..3 of column l of the 4 x 16 block whose row l / 4,
// columns 4 (l % 4) .. + 3, its address names.
__device__ __forceinline__ f16x4 read_transposed(const _Float16 *at) {
  const i16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4 *)(at));
  return __builtin_bit_cast(f16x4, r);
}
__device__ __forceinline__ f16x8 join(f16x4 a, f16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}
// The sums of hi hi' and of hi lo' + lo hi', which are kLo times as large.
struct Sum {
  f32x16 hh = zero16(), cross = zero16();
  __device__ __forceinline__ float operator[](int e) const { return hh[e] + cross[e] * (1.f / kLo); }
};
__device__ __forceinline__ void product(f16x8 a, f16x8 b, f32x16 &acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void product3(f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl, Sum &acc) {
  product(ah, bl, acc.cross);
  product(ah, bh, acc.hh);
  product(al, bh, acc.cross);
}

// ----------------------------------------------------------------------------- norm and first y
// The update before normalisation.  `first`: the momentum is still the old one and is written.
__device__ __forceinline__ float update_value(const NsParams &p, long long at, bool first) {
  const float x = p.x[at];
  if (!p.m) return x;
  const float gs = p.grad_scale * x;
  float m = p.m[at];
  if (first) {
    m = p.momentum * m + gs;
    p.m[at] = m;
  }
  return p.nesterov ? gs + p.momentum * m : m;
}
__device__ __forceinline__ f32x4 update_quad(const NsParams &p, long long at, bool first) {
  const f32x4 x = *reinterpret_cast<const f32x4 *>(p.x + at);
  if (!p.m) return x;
  f32x4 m = *reinterpret_cast<const f32x4 *>(p.m + at), u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float gs = p.grad_scale * x[e];
    if (first) m[e] = p.momentum * m[e] + gs;
    u[e] = p.nesterov ? gs + p.momentum * m[e] : m[e];
  }
  if (first) *reinterpret_cast<f32x4 *>(p.m + at) = m;
  return u;
}

__device__ __forceinline__ double wave_sum(double s) {
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  return s;
}

// Sum of squares of one matrix in PARTS parts in a fixed order; Muon: the new momentum (255 MB: 50 us).
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsParams p) {
  __shared__ double red[4];
  const int part = blockIdx.x % PARTS;
  const long long k = blockIdx.x / PARTS;
  const long long size = (long long)p.rows * p.cols, chunk = ((size + PARTS - 1) / PARTS + 3) / 4 * 4;
  const long long begin = part * chunk < size ? part * chunk : size;
  const long long end = begin + chunk < size ? begin + chunk : size;
  double s = 0.0;
  if (p.flat) {
    const long long quads = (end - begin) / 4;
#pragma unroll 4
    for (long long i = threadIdx.x; i < quads; i += 256) {
      const f32x4 u = update_quad(p, k * p.stride_x + begin + 4 * i, true);
#pragma unroll
      for (int e = 0; e < 4; ++e) s += (double)u[e] * (double)u[e];
    }
    const long long i = begin + 4 * quads + threadIdx.x;
    if (i < end) {
      const float u = update_value(p, k * p.stride_x + i, true);
      s += (double)u * (double)u;
    }
  } else {
    long long i = begin + threadIdx.x, row = i / p.cols;
    int col = (int)(i - row * p.cols);
    const int step_rows = 256 / p.cols, step_cols = 256 % p.cols;
    for (; i < end; i += 256) {
      const float u = update_value(p, k * p.stride_x + row * p.ld_x + col, true);
      s += (double)u * (double)u;
      row += step_rows, col += step_cols;
      if (col >= p.cols) col -= p.cols, ++row;
    }
  }
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) p.sums[k * PARTS + part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Element (i, j) of the r x n form is element (i, j) or, tall, (j, i) of the user's matrix.
__device__ __forceinline__ void emit(const NsParams &p, long long k, int i, int j, float v) {
  if (i >= p.r || j >= p.n) return;
  const long long at = k * p.stride_out + (p.tall ? j * p.ld_out + i : i * p.ld_out + j);
  if (p.p)
    p.p[at] = p.p[at] * p.keep - p.step * v;
  else
    p.out[at] = v;
}
// Four neighbouring elements (row, col ..) of the user's matrix; `old`: the parameter, loaded before (p.vec).
__device__ __forceinline__ f32x4 emit_old(const NsParams &p, long long k, int row, int col) {
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (p.p && p.vec && row < p.rows && col + 3 < p.cols)
    x = *reinterpret_cast<const f32x4 *>(p.p + k * p.stride_out + row * p.ld_out + col);
  return x;
}
__device__ __forceinline__ void emit4(const NsParams &p, long long k, int row, int col, f32x4 v, f32x4 old) {
  if (row >= p.rows) return;
  const long long at = k * p.stride_out + row * p.ld_out + col;
  if (p.vec && col + 3 < p.cols) {
    if (p.p) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = old[e] * p.keep - p.step * v[e];
      *reinterpret_cast<f32x4 *>(p.p + at) = v;
    } else {
      *reinterpret_cast<f32x4 *>(p.out + at) = v;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.cols) {
      if (p.p)
        p.p[at + e] = p.p[at + e] * p.keep - p.step * v[e];
      else
        p.out[at + e] = v[e];
    }
}

// y = u / (|u| + eps) with its planes, one 64 x 64 tile per workgroup; `last`: only the result.
__global__ __launch_bounds__(256) void ns_start_kernel(const NsParams p, int last) {
  constexpr int T = 64;
  __shared__ float tile[T][T + 1];
  const int tj = p.np / T, tiles = (p.rp / T) * tj;
  const long long k = blockIdx.x / tiles;
  const int t = blockIdx.x % tiles, i0 = t / tj * T, j0 = t % tj * T;
  const float norm = (float)sqrt(wave_sum(p.sums[k * PARTS + (threadIdx.x & 63)])) + p.eps;
  if (p.tall) {  // rows of the user's matrix are columns here
    float x[T * T / 256];
#pragma unroll
    for (int w = 0; w < T * T / 256; ++w) {
      const int u = threadIdx.x + 256 * w, j = min(j0 + u / T, p.n - 1), i = min(i0 + u % T, p.r - 1);
      x[w] = update_value(p, k * p.stride_x + j * p.ld_x + i, false);
    }
#pragma unroll
    for (int w = 0; w < T * T / 256; ++w) {
      const int u = threadIdx.x + 256 * w, j = u / T, i = u % T;
      tile[i][j] = i0 + i < p.r && j0 + j < p.n ? x[w] / norm : 0.f;
    }
    __syncthreads();
  }
#pragma unroll
  for (int w = 0; w < T * T / 4 / 256; ++w) {
    const int u = threadIdx.x + 256 * w, i = u / (T / 4), j = u % (T / 4) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (p.tall) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = tile[i][j + e];
    } else if (i0 + i < p.r) {
      const long long at = k * p.stride_x + (i0 + i) * p.ld_x + j0 + j;
      if (p.flat && p.cols % 4 == 0) {
        if (j0 + j < p.n) v = update_quad(p, at, false);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j0 + j + e < p.n) v[e] = update_value(p, at + e, false);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + j + e < p.n) v[e] /= norm;
    }
    if (last) {
      if (p.tall) {
#pragma unroll
        for (int e = 0; e < 4; ++e) emit(p, k, i0 + i, j0 + j + e, v[e]);
      } else {
        emit4(p, k, i0 + i, j0 + j, v, emit_old(p, k, i0 + i, j0 + j));
      }
      continue;
    }
    const long long row = k * p.rp + i0 + i;
    store_split4(p.yp[0] + plane_at(row, j0 + j, p.np), v, kY);
  }
}

// --------------------------------------------------------------------------------------- products
enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

// C[i][j] = sum_k P[i][k] Q[j][k]:
//   GRAM: P = Q = y      -> g and its planes
//   POLY: P = Q = g      -> planes of b g + c g g
//   APPLY: P = that, Q = y^T -> y = a y + C with its planes;  LAST: the same, result to the user's matrix
// What else goes into four neighbouring elements (i, j..j+3), y or g: parts loaded before the sums are needed.
struct Parts {
  f16x4 hi, lo;
};
template <int MODE>
__device__ __forceinline__ Parts addend(const NsParams &p, int flip, long long k, int i, int j) {
  if constexpr (MODE == GRAM) return Parts{};
  const _Float16 *at = MODE == POLY ? p.gp + plane_at(k * p.rp + i, j, p.rp) : p.yp[flip] + plane_at(k * p.rp + i, j, p.np);
  return Parts{*reinterpret_cast<const f16x4 *>(at), *reinterpret_cast<const f16x4 *>(at + 32)};
}
// The value of these elements, stored as planes (LAST: not stored).
template <int MODE>
__device__ __forceinline__ f32x4 finish(const NsParams &p, int flip, long long k, int i, int j, f32x4 acc, Parts add) {
  const long long row = k * p.rp + i;
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = (float)add.hi[e] + (float)add.lo[e] * (1.f / kLo);
    if constexpr (MODE == GRAM)
      v[e] = acc[e] * (1.f / (kY * kY));
    else if constexpr (MODE == POLY)
      v[e] = p.b * (x * (1.f / kG)) + p.c * (acc[e] * (1.f / (kG * kG)));
    else
      v[e] = p.a * (x * (1.f / kY)) + acc[e] * (1.f / (kG * kY));
  }
  if constexpr (MODE == GRAM) store_split4(p.gp + plane_at(row, j, p.rp), v, kG);
  if constexpr (MODE == POLY) store_split4(p.bp + plane_at(row, j, p.rp), v, kG);
  if constexpr (MODE == APPLY) store_split4(p.yp[1 - flip] + plane_at(row, j, p.np), v, kY);
  return v;
}
// Four neighbouring elements (j, i..i+3) of the transposed tile: the mirrored part of a symmetric product, or the
// result of a tall matrix.
template <int MODE>
__device__ __forceinline__ void finish_transposed(const NsParams &p, long long k, int j, int i, f32x4 v) {
  if constexpr (MODE == LAST)
    emit4(p, k, j, i, v, emit_old(p, k, j, i));
  else
    store_split4((MODE == GRAM ? p.gp : p.bp) + plane_at(k * p.rp + j, i, p.rp), v, kG);
}

// Tile t of a list: all tiles column by column (a column of tiles shares the long operand, and all of them the
// short one), or those on and below the diagonal.
template <bool LOWER>
__device__ __forceinline__ void tile_of(int t, int ti, int &i, int &j) {
  if constexpr (LOWER) {
    i = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    j = t - i * (i + 1) / 2;
  } else {
    j = t / ti;
    i = t - j * ti;
  }
}

// 16 bytes at base + voff + soff (bytes): a scalar base and offset, so that a thread keeps one address per operand.
__device__ __forceinline__ f16x8 load_unit(const _Float16 *base, int voff, int soff) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16 *>(base), 0, 0x7fffffff, 0x00020000);
  return __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}

// T x T tiles, NW waves of T/2 x 2T/NW each, slabs of 32 k double-buffered in LDS and DIST more of them on
// their way in registers: a slab is 768 cycles of matrix work at T = 128, what another XCD wrote is
// 2000 to 3000 cycles away.
// The workgroups of an XCD (every eighth) take neighbouring tiles, so that they share operands in its L2.
template <int MODE, int T, int NW>
__global__ __launch_bounds__(64 * NW, 4) void ns_tile_kernel(const NsParams p, int flip, int total) {
  constexpr bool LOWER = MODE <= POLY, TR = MODE >= APPLY;
  constexpr int NX = T / 64, NY = 2 * T / NW / 32;  // 32-wide blocks of a wave in each direction
  constexpr int UNITS = T * 8;                      // 16-byte units of an operand's slab
  constexpr int THREADS = 64 * NW, LOADS = UNITS / THREADS;
  constexpr int DIST = 2;
  constexpr int SP = T + 4;  // pitch of the sums in the epilogue
  constexpr int LDS_BYTES = T * SP * 4 > 4 * UNITS * 16 ? T * SP * 4 : 4 * UNITS * 16;
  __shared__ __attribute__((aligned(16))) char lds_bytes[LDS_BYTES];
  f16x8 (*lds)[2][UNITS] = reinterpret_cast<f16x8 (*)[2][UNITS]>(lds_bytes);  // [buffer][operand]
  float *sums = reinterpret_cast<float *>(lds_bytes);
  const int per = (total + 7) / 8, id = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (id >= total || (int)blockIdx.x / 8 >= per) return;
  const int cols = TR ? p.np : p.rp, depth = MODE == GRAM ? p.np : p.rp;
  const int ti = p.rp / T, tj = cols / T, tiles = LOWER ? ti * (ti + 1) / 2 : ti * tj;
  const long long k = id / tiles;
  int bi, bj;
  tile_of<LOWER>(id % tiles, ti, bi, bj);
  const int i0 = bi * T, j0 = bj * T;
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5, wave = threadIdx.x >> 6;
  const int wi = (wave & 1) * (T / 2), wj = (wave >> 1) * (32 * NY);

  // Operand slabs: THREADS / 8 rows of P (and Q) per pass, or, transposed, 4 THREADS / T rows of T columns.
  // A unit's place in LDS is its own XOR a number of its row that spreads what one read touches over the banks:
  // 16 rows of one unit, or, transposed, four rows of four neighbouring units.
  const _Float16 *P = (MODE == GRAM ? p.yp[flip] : MODE == POLY ? p.gp : p.bp) + (k * p.rp + i0) * 2ll * depth;
  const _Float16 *Q = MODE == POLY ? p.gp : p.yp[flip];
  Q += TR ? k * p.rp * 2ll * cols + 2 * j0 : (k * p.rp + j0) * 2ll * depth;
  const int prow = threadIdx.x / 8, punit = threadIdx.x % 8, qrow = threadIdx.x / (T / 4), qunit = threadIdx.x % (T / 4);
  const int pv = (prow * 2 * depth + punit * 8) * 2, qv = TR ? (qrow * 2 * cols + qunit * 8) * 2 : pv;
  const int ppass = (THREADS / 8) * 2 * depth * 2, qpass = TR ? (4 * THREADS / T) * 2 * cols * 2 : ppass;
  auto row_swizzle = [](int row) { return (row >> 1) & 7; };
  auto tr_swizzle = [](int row) { return (row & 3) * 4; };
  const int pd = prow * 8 + (punit ^ row_swizzle(prow));
  const int qd = TR ? qrow * (T / 4) + (qunit ^ tr_swizzle(qrow)) : pd;
  const long long qslab = TR ? 32ll * 2 * cols : 64;

  Sum acc[NX][NY];
  f16x8 pr[DIST][LOADS], qr[DIST][LOADS];
  const int slabs = depth / 32;
  auto fetch = [&](int s, f16x8 (&x)[LOADS], f16x8 (&y)[LOADS]) {
    s = min(s, slabs - 1);  // (behind the end: loaded and not used)
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      x[u] = load_unit(P + s * 64ll, pv, u * ppass);
      y[u] = load_unit(Q + s * qslab, qv, u * qpass);
    }
  };
  auto put = [&](int buf, const f16x8 (&x)[LOADS], const f16x8 (&y)[LOADS]) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      lds[buf][0][pd + THREADS * u] = x[u];
      lds[buf][1][qd + THREADS * u] = y[u];
    }
  };
#pragma unroll
  for (int d = 0; d < DIST; ++d) fetch(d, pr[d], qr[d]);
  put(0, pr[0], qr[0]);
  fetch(DIST, pr[0], qr[0]);
  __syncthreads();
  // slab s is in LDS, slabs s + 1 .. s + DIST are on their way, slab t in registers t % DIST.  The body has no
  // branch: where loads may or may not have been issued the compiler waits for all of them.
  auto multiply = [&](int s, int h) {
    const f16x8 *lp = lds[s & 1][0], *lq = lds[s & 1][1];
    // blocks of P (columns of the result tile's MFMA form) and of Q
    auto read_p = [&](int part, f16x8 (&to)[NX]) {
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const int row = wi + 32 * x + c;
        to[x] = lp[row * 8 + ((4 * part + 2 * h + g) ^ row_swizzle(row))];
      }
    };
    auto read_q = [&](int part, f16x8 (&to)[NY]) {
#pragma unroll
      for (int y = 0; y < NY; ++y) {
        if constexpr (TR) {
          const int sub = (lane >> 4) & 1, k0 = 16 * h + 8 * g + ((lane & 15) >> 2);
          const int unit = ((wj >> 5) + y) * 8 + 4 * part + 2 * sub + ((lane & 3) >> 1);
          const _Float16 *base = reinterpret_cast<const _Float16 *>(lq) + 4 * (lane & 1);
          to[y] = join(read_transposed(base + (k0 * (T / 4) + (unit ^ tr_swizzle(k0))) * 8),
                       read_transposed(base + ((k0 + 4) * (T / 4) + (unit ^ tr_swizzle(k0 + 4))) * 8));
        } else {
          const int row = wj + 32 * y + c;
          to[y] = lq[row * 8 + ((4 * part + 2 * h + g) ^ row_swizzle(row))];
        }
      }
    };
    // the sums of all blocks in turn, operands in the order of their use: registers are short
    f16x8 ph[NX], pl[NX], qh[NY], ql[NY];
    read_p(0, ph), read_q(0, qh), read_q(1, ql), read_p(1, pl);
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int y = 0; y < NY; ++y) product(qh[y], ph[x], acc[x][y].hh);
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int y = 0; y < NY; ++y) product(ql[y], ph[x], acc[x][y].cross);
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int y = 0; y < NY; ++y) product(qh[y], pl[x], acc[x][y].cross);
  };
  auto step = [&](int s, f16x8 (&x)[LOADS], f16x8 (&y)[LOADS]) {
    multiply(s, 0);
    put((s + 1) & 1, x, y);
    fetch(s + 1 + DIST, x, y);
    multiply(s, 1);
    __syncthreads();
  };
  int s0 = 0;
  for (; s0 + DIST <= slabs; s0 += DIST)
#pragma unroll
    for (int d = 0; d < DIST; ++d) step(s0 + d, pr[(d + 1) % DIST], qr[(d + 1) % DIST]);
#pragma unroll
  for (int d = 0; d + 1 < DIST; ++d)
    if (s0 + d < slabs) step(s0 + d, pr[(d + 1) % DIST], qr[(d + 1) % DIST]);
  // Epilogue by way of LDS, so that rows are read and written 512 bytes at a time.  Register 4 q + e of lane (c, g)
  // is element (i = c, j = 8 q + 4 g + e) of a block.
  constexpr int QUADS = T * T / 4 / THREADS, RQ = T / 4;  // quads of a thread, of a row
  Parts add[QUADS];
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int quad = threadIdx.x + THREADS * u;
    add[u] = addend<MODE>(p, flip, k, i0 + quad / RQ, j0 + quad % RQ * 4);
  }
#pragma unroll
  for (int x = 0; x < NX; ++x)
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[x][y][4 * q + e];
        *reinterpret_cast<f32x4 *>(sums + (wi + 32 * x + c) * SP + wj + 32 * y + 8 * q + 4 * g) = v;
      }
  __syncthreads();
  const bool turn = LOWER ? bi != bj : MODE == LAST && p.tall;  // (uniform)
  f32x4 old[MODE == LAST ? QUADS : 1];
  if constexpr (MODE == LAST) {
#pragma unroll
    for (int u = 0; u < QUADS; ++u) {
      const int quad = threadIdx.x + THREADS * u;
      if (!turn) old[u] = emit_old(p, k, i0 + quad / RQ, j0 + quad % RQ * 4);
    }
  }
#pragma unroll
  for (int u = 0; u < QUADS; ++u) {
    const int quad = threadIdx.x + THREADS * u, i = quad / RQ, j = quad % RQ * 4;
    f32x4 *at = reinterpret_cast<f32x4 *>(sums + i * SP + j);
    const f32x4 v = finish<MODE>(p, flip, k, i0 + i, j0 + j, *at, add[u]);
    if (turn)
      *at = v;
    else if constexpr (MODE == LAST)
      emit4(p, k, i0 + i, j0 + j, v, old[u]);
  }
  if (!turn) return;
  __syncthreads();
  for (int block = threadIdx.x; block < RQ * RQ; block += THREADS) {  // 4 x 4 blocks, lanes along i
    const int i = block % RQ * 4, j = block / RQ * 4;
    f32x4 r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const f32x4 *>(sums + (i + e) * SP + j);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      finish_transposed<MODE>(p, k, j0 + j + e, i0 + i, f32x4{r[0][e], r[1][e], r[2][e], r[3][e]});
  }
}

// 32 x 32 tiles, the contraction dealt to NW waves, operands straight from memory: the step of y of 257 x 1000 takes
// 7.5 us (288 workgroups), mostly round trips to memory.
template <int MODE, int NW>
__global__ __launch_bounds__(64 * NW) void ns_small_kernel(const NsParams p, int flip, int ti) {
  constexpr bool LOWER = MODE <= POLY, TR = MODE >= APPLY;
  constexpr int U = TR ? 4 : 8;       // steps of 16 k in flight
  constexpr int PITCH = 80;           // fp16 pitch of a row of transposed operand (64 + a shift of 32 bytes)
  constexpr int SUM_PITCH = 36, REGION = TR ? 2 * 16 * PITCH * 2 : 32 * SUM_PITCH * 4;  // bytes of a wave
  static_assert(REGION >= 32 * SUM_PITCH * 4, "the wave's sums go where its operand was");
  __shared__ __attribute__((aligned(16))) char lds[NW][REGION];
  const int cols = TR ? p.np : p.rp, depth = MODE == GRAM ? p.np : p.rp;
  const int tj = TR ? (p.n + 31) / 32 : ti, tiles = LOWER ? ti * (ti + 1) / 2 : ti * tj;
  const long long k = blockIdx.x / tiles;
  int bi, bj;
  tile_of<LOWER>(blockIdx.x % tiles, ti, bi, bj);
  const int i0 = bi * 32, j0 = bj * 32;
  const _Float16 *P = MODE == GRAM ? p.yp[flip] : MODE == POLY ? p.gp : p.bp;
  const _Float16 *Q = MODE == GRAM ? p.yp[flip] : MODE == POLY ? p.gp : p.yp[flip];
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = ((MODE == GRAM ? p.n : p.r) + 15) / 16, share = (steps + NW - 1) / NW;  // k behind n / r is padding
  const int s0 = min(wave * share, steps), s1 = min(s0 + share, steps);
  const _Float16 *prow = P + (k * p.rp + i0 + c) * 2ll * depth + 8 * g;
  const _Float16 *qrow = TR ? Q + (k * p.rp + (lane >> 2)) * 2ll * cols + 2 * j0 + 8 * (lane & 3)
                            : Q + (k * p.rp + j0 + c) * 2ll * depth + 8 * g;
  const int i = threadIdx.x >> 3, j = (threadIdx.x & 7) * 4;  // this thread's elements of the result
  Parts add = {};
  if (threadIdx.x < 256) add = addend<MODE>(p, flip, k, i0 + i, j0 + j);
  Sum acc;
  [[maybe_unused]] _Float16 *qt = reinterpret_cast<_Float16 *>(lds[wave]);
  for (int s = s0; s < s1; s += U) {
    f16x8 a[U][2], b[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(s + u, s1 - 1), off = (t >> 1) * 64 + (t & 1) * 16;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        a[u][part] = *reinterpret_cast<const f16x8 *>(prow + off + 32 * part);
        if constexpr (TR)
          b[u][part] = *reinterpret_cast<const f16x8 *>(qrow + t * 16ll * 2 * cols + 32 * part);
        else
          b[u][part] = *reinterpret_cast<const f16x8 *>(qrow + off + 32 * part);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // keep them all in flight
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u >= s1) a[u][0] = a[u][1] = f16x8{};  // (a step that was loaded twice adds nothing)
    if constexpr (TR) {  // through the wave's own part of LDS, two steps at a time (so that three workgroups fit a CU)
#pragma unroll
      for (int u = 0; u < U; u += 2) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int part = 0; part < 2; ++part)
            *reinterpret_cast<f16x8 *>(qt + (x * 16 + (lane >> 2)) * PITCH + 32 * part + 8 * (lane & 3)) = b[u + x][part];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const int row = x * 16 + 8 * g + ((lane & 15) >> 2), col = 32 * part + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            b[u + x][part] = join(read_transposed(qt + row * PITCH + col), read_transposed(qt + (row + 4) * PITCH + col));
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) product3(b[u][0], b[u][1], a[u][0], a[u][1], acc);
  }
  float *own = reinterpret_cast<float *>(lds[wave]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[4 * q + e];
    *reinterpret_cast<f32x4 *>(own + c * SUM_PITCH + 8 * q + 4 * g) = v;
  }
  __syncthreads();
  const bool mine = threadIdx.x < 256;  // has elements of the result
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (mine) {
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const f32x4 w = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(lds[x]) + i * SUM_PITCH + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += w[e];
    }
    v = finish<MODE>(p, flip, k, i0 + i, j0 + j, v, add);
  }
  if (LOWER ? bi != bj : MODE == LAST && p.tall) {
    __syncthreads();
    float *turn = reinterpret_cast<float *>(lds[0]);
    if (mine) *reinterpret_cast<f32x4 *>(turn + i * SUM_PITCH + j) = v;
    __syncthreads();
    if (!mine) return;
    f32x4 w;  // (j0 + i, i0 + j ..)
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = turn[(j + e) * SUM_PITCH + i];
    finish_transposed<MODE>(p, k, j0 + i, i0 + j, w);
  } else if constexpr (MODE == LAST) {
    if (mine) emit4(p, k, i0 + i, j0 + j, v, emit_old(p, k, i0 + i, j0 + j));
  }
}

// The symmetric products where 32 x 32 tiles leave half of the CUs without work: 16 x 16 tiles, half as much for each to read.
// The contraction is dealt to the waves, 32 k a step, a line of planes for 16 rows; the first wave adds the sums.
// 257 x 1000: y y^T 6.6 us, the polynomial 4.7 (32 x 32 tiles: 10.8 and 6.2).
template <int MODE, int NW>
__global__ __launch_bounds__(64 * NW) void ns_lower_kernel(const NsParams p, int flip, int ti) {
  static_assert(MODE <= POLY, "the symmetric products");
  constexpr int U = 4, PITCH = 20;  // steps in flight
  __shared__ __attribute__((aligned(16))) float lds[NW][16 * PITCH];
  const int depth = MODE == GRAM ? p.np : p.rp, tiles = ti * (ti + 1) / 2;
  const long long k = blockIdx.x / tiles;
  int bi, bj;
  tile_of<true>(blockIdx.x % tiles, ti, bi, bj);
  const int i0 = bi * 16, j0 = bj * 16;
  const _Float16 *P = MODE == GRAM ? p.yp[flip] : p.gp;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = ((MODE == GRAM ? p.n : p.r) + 31) / 32, share = (steps + NW - 1) / NW;  // what is behind is zero
  const int s0 = min(wave * share, steps), s1 = min(s0 + share, steps);
  const _Float16 *prow = P + (k * p.rp + i0 + c) * 2ll * depth + 8 * g;
  const _Float16 *qrow = P + (k * p.rp + j0 + c) * 2ll * depth + 8 * g;
  const int i = lane >> 2, j = (lane & 3) * 4;  // the first wave's elements of the result
  Parts add = {};
  if (wave == 0) add = addend<MODE>(p, flip, k, i0 + i, j0 + j);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f}, cross = acc;
  for (int s = s0; s < s1; s += U) {
    f16x8 a[U][2], b[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const int at = min(s + u, s1 - 1) * 64 + 32 * part;
        a[u][part] = *reinterpret_cast<const f16x8 *>(prow + at);
        b[u][part] = *reinterpret_cast<const f16x8 *>(qrow + at);
      }
    __builtin_amdgcn_sched_barrier(0);  // keep them all in flight
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= s1) a[u][0] = a[u][1] = f16x8{};  // (a step that was loaded twice adds nothing)
      cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[u][0], a[u][1], cross, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[u][0], a[u][0], acc, 0, 0, 0);
      cross = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[u][1], a[u][0], cross, 0, 0, 0);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] += cross[e] * (1.f / kLo);
  *reinterpret_cast<f32x4 *>(lds[wave] + c * PITCH + 4 * g) = acc;
  __syncthreads();
  if (wave > 0) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < NW; ++x) {
    const f32x4 w = *reinterpret_cast<const f32x4 *>(lds[x] + i * PITCH + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += w[e];
  }
  v = finish<MODE>(p, flip, k, i0 + i, j0 + j, v, add);
  if (bi == bj) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  *reinterpret_cast<f32x4 *>(lds[0] + i * PITCH + j) = v;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  f32x4 w;  // (j0 + i, i0 + j ..)
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = lds[0][(j + e) * PITCH + i];
  finish_transposed<MODE>(p, k, j0 + i, i0 + j, w);
}

// Both sides <= 128: everything in one launch.  Sixteen waves, one 32 x 32 block of g and of y each; the planes of
// y and of g, then b g + c g g, are in LDS (70 KiB each), what a wave adds to its products in registers.  All
// blocks of g are computed: writing a block's mirror image, two bytes at a time, takes longer than its product.
// 96 x 96, five steps: 27 us, 1.4 a product: operands from LDS 0.7, matrix cores 0.7, one after the other.
// A row of planes takes 3 mod 16 units of 16 bytes, so that 16 rows of one unit, and mostly four rows of four
// neighbouring ones, are on different banks.
constexpr int ONE_WAVES = 16;
__host__ __device__ constexpr int one_pitch(int blocks) { return 8 * blocks + (blocks % 2 ? 11 : 3); }
__global__ __launch_bounds__(64 * ONE_WAVES) void ns_one_kernel(const NsParams p) {
  extern __shared__ __attribute__((aligned(16))) f16x8 one_lds[];
  __shared__ double red[ONE_WAVES];
  const int tr = (p.r + 31) / 32, tn = (p.n + 31) / 32;  // blocks of 32 in use
  const int yp = one_pitch(tn), gp = one_pitch(tr);
  f16x8 *yl = one_lds, *gl = one_lds + tr * 32 * yp;  // [row][column block][8 units]
  int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long k = blockIdx.x;
  // this wave's block of y and of g
  const int yi = wave / tn, yj = wave % tn, gi = wave / tr, gj = wave % tr;
  const bool y_mine = yi < tr, g_mine = gi < tr;
  float y[16];  // behind the norm: times kY
  double s = 0.0;
  // Element e of the lane: row 32 yi + c, column 32 yj + 4 g + 8 (e / 4) + e % 4.  Every load is issued, its place
  // clamped: a branch around each would wait for one after the other (96 x 96 without a step: 11 us instead of 6).
  const int row = 32 * yi + c, col = 32 * yj + 4 * g;
  const bool quads = p.flat && !p.tall && p.cols % 4 == 0;
  {
    const long long si = p.tall ? 1 : p.ld_x, sj = p.tall ? p.ld_x : 1;
    const long long line = k * p.stride_x + min(row, p.r - 1) * si;
    auto load = [&](const float *x, float (&v)[16]) {
      if (quads) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 w = *reinterpret_cast<const f32x4 *>(x + line + min(col + 8 * q, p.n - 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * q + e] = w[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = x[line + min(col + 8 * (e / 4) + e % 4, p.n - 1) * sj];
      }
    };
    load(p.x, y);
    if (p.m) {
      float m[16];
      load(p.m, m);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float gs = p.grad_scale * y[e];
        m[e] = p.momentum * m[e] + gs;
        y[e] = p.nesterov ? gs + p.momentum * m[e] : m[e];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int j = col + 8 * (e / 4) + e % 4;
        if (row < p.r && j < p.n) p.m[line + j * sj] = m[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (row >= p.r || col + 8 * (e / 4) + e % 4 >= p.n) y[e] = 0.f;
      s += (double)y[e] * (double)y[e];
    }
  }
  s = wave_sum(s);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < ONE_WAVES; ++w) s += red[w];
  const float norm = (float)sqrt(s) + p.eps;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (row < p.r && col + 8 * (e / 4) + e % 4 < p.n) y[e] = y[e] / norm * kY;
  // block (bi, bj) of a matrix with `blocks` column blocks, from the registers' layout
  auto store = [&](f16x8 *m, int pitch, int bi, int bj, const float (&x)[16], float scale) {
    const int row = 32 * bi + c;
    _Float16 *line = reinterpret_cast<_Float16 *>(m + row * pitch + bj * 8);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f16x4 hi, lo;
      split4(f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]}, scale, hi, lo);
      *reinterpret_cast<f16x4 *>(line + 8 * q + 4 * g) = hi;
      *reinterpret_cast<f16x4 *>(line + 8 * (4 + q) + 4 * g) = lo;
    }
  };
  struct Operand {
    f16x8 part[2];  // of 16 k
  };
  // row 32 block + c, columns 16 t .. + 15
  auto rows = [&](const f16x8 *m, int pitch, int block, int t) {
    const f16x8 *at = m + (32 * block + c) * pitch + 8 * (t >> 1) + 2 * (t & 1) + g;
    return Operand{{at[0], at[4]}};
  };
  // column 32 cb + c of y, rows 16 t .. + 15
  auto columns = [&](int t, int cb) {
    Operand o;
    const _Float16 *at = reinterpret_cast<const _Float16 *>(yl + (16 * t + 8 * g + ((lane & 15) >> 2)) * yp + 8 * cb) +
                         16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
    for (int part = 0; part < 2; ++part)
      o.part[part] = join(read_transposed(at + 32 * part), read_transposed(at + 4 * yp * 8 + 32 * part));
    return o;
  };
  // sum over `blocks` times 32 k; the next operands are on their way behind each product.  (The first product is
  // written out: it takes constants where the others take the registers of the sums.)
  auto contract = [&](int blocks, auto left, auto right) {
    Sum acc;
    auto multiply = [&](const Operand &a, const Operand &b) { product3(a.part[0], a.part[1], b.part[0], b.part[1], acc); };
    Operand a0 = left(0), b0 = right(0), a1 = left(1), b1 = right(1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(a0, b0);
#pragma unroll 1
    for (int t = 2; t < 2 * blocks; t += 2) {
      a0 = left(t), b0 = right(t);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a1, b1);
      a1 = left(t + 1), b1 = right(t + 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(a0, b0);
    }
    multiply(a1, b1);
    return acc;
  };
  // of row blocks bi and bj of one matrix
  auto symmetric = [&](const f16x8 *m, int pitch, int blocks, int bi, int bj) {
    return contract(blocks, [&](int t) { return rows(m, pitch, bj, t); }, [&](int t) { return rows(m, pitch, bi, t); });
  };
  if (p.steps > 0 && y_mine) store(yl, yp, yi, yj, y, 1.f);
  __syncthreads();
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    // (the compiler would compute every address of the body before the loop and run out of registers)
    asm volatile("" : "+v"(lane), "+v"(c), "+v"(g));
    float v[16];  // g times kY^2
    if (g_mine) {  // g = y y^T
      const Sum acc = symmetric(yl, yp, tn, gi, gj);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[e];
      store(gl, gp, gi, gj, v, kG / (kY * kY));
    }
    __syncthreads();
    if (g_mine) {  // b g + c g g
      const Sum acc = symmetric(gl, gp, tr, gi, gj);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = p.b * (1.f / (kY * kY)) * v[e] + p.c * (1.f / (kG * kG)) * acc[e];
    }
    __syncthreads();
    if (g_mine) store(gl, gp, gi, gj, v, kG);
    __syncthreads();
    if (y_mine) {  // y = a y + that y
      const Sum acc = contract(tr, [&](int t) { return columns(t, yj); }, [&](int t) { return rows(gl, gp, yi, t); });
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = p.a * y[e] + acc[e] * (1.f / kG);
    }
    if (step + 1 < p.steps) {
      __syncthreads();
      if (y_mine) store(yl, yp, yi, yj, y, 1.f);
      __syncthreads();
    }
  }
  if (row >= p.r) return;
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] *= 1.f / kY;
  const long long si = p.tall ? 1 : p.ld_out, sj = p.tall ? p.ld_out : 1, line = k * p.stride_out + row * si;
  if (p.vec && !p.tall && p.cols % 4 == 0) {
    f32x4 old[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (p.p) old[q] = *reinterpret_cast<const f32x4 *>(p.p + line + min(col + 8 * q, p.n - 4));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p.p ? old[q][e] * p.keep - p.step * y[4 * q + e] : y[4 * q + e];
      if (col + 8 * q < p.n) *reinterpret_cast<f32x4 *>((p.p ? p.p : p.out) + line + col + 8 * q) = v;
    }
    return;
  }
  if (p.p) {
    float old[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) old[e] = p.p[line + min(col + 8 * (e / 4) + e % 4, p.n - 1) * sj];
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = old[e] * p.keep - p.step * y[e];
  }
  float *to = p.p ? p.p : p.out;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int j = col + 8 * (e / 4) + e % 4;
    if (j < p.n) to[line + j * sj] = y[e];
  }
}

// ------------------------------------------------------------------------------------------- plan
enum { FORM_ONE, FORM_SMALL, FORM_64, FORM_128 };

long long padded(long long x, int t) { return (x + t - 1) / t * t; }

int plan_form(int r, int n, int batch) {
  if (n <= ONE) return FORM_ONE;
  const long long enough = vitk::cu_count() * 3 / 4;
  if (batch * (padded(r, 128) / 128) * (padded(n, 128) / 128) >= enough) return FORM_128;
  if (batch * (padded(r, 64) / 64) * (padded(n, 64) / 64) >= enough) return FORM_64;
  return FORM_SMALL;
}

// Workspace of one call: sums, then the planes (4 bytes an element).
size_t plan(NsParams *p, float *workspace, int *form) {
  p->tall = p->rows > p->cols;
  p->r = p->tall ? p->cols : p->rows;
  p->n = p->tall ? p->rows : p->cols;
  *form = plan_form(p->r, p->n, p->batch);
  if (*form == FORM_ONE) return 0;
  const int t = *form == FORM_128 ? 128 : 64;
  p->rp = (int)padded(p->r, t);
  p->np = (int)padded(p->n, t);
  const size_t b = p->batch, yy = b * p->rp * p->np, gg = b * p->rp * p->rp;
  char *at = reinterpret_cast<char *>(workspace);
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char *r = at ? at + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return r;
  };
  p->sums = reinterpret_cast<double *>(take(b * PARTS * sizeof(double)));
  for (auto *planes : {&p->yp[0], &p->yp[1]}) *planes = reinterpret_cast<_Float16 *>(take(yy * 4));
  for (auto *planes : {&p->gp, &p->bp}) *planes = reinterpret_cast<_Float16 *>(take(gg * 4));
  return used;
}

bool size_ok(int64_t rows, int64_t cols, int64_t batch) {
  return rows >= 0 && cols >= 0 && batch >= 0 && rows <= (1 << 20) && cols <= (1 << 20);
}

// Does the iteration t -> a t + b t^3 + c t^5 stay where the fixed scales hold?  From |t| <= top, the largest values
// of the odd polynomial, and of b q + c q^2 with q = t^2, are at the ends or where their derivatives vanish.  Rounding
// may carry a value over an end, and a polynomial that is steep there carries it on and out of the range within
// a few steps (5 t - 20 t^3 + 16 t^5 multiplies what is above 1 by 25), so each step starts from 2^-14 more: sums of
// 16384 terms are not off by as much.
constexpr double SLACK = 1.0 + 1.0 / 16384;
bool bounded(double a, double b, double c, int steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double top = SLACK;
  for (int s = 0; s < steps; ++s) {
    // the roots of a + 3 b q + 5 c q^2 without a difference of neighbours (c may be tiny, or 0: then one of them is
    // an infinity, whose place the end takes, or no number)
    const double end = top * top, root = std::sqrt(std::max(9.0 * b * b - 20.0 * a * c, 0.0));
    const double t = -0.5 * (3.0 * b + std::copysign(root, b));
    const double at[] = {end, -b / (2.0 * c), t / (5.0 * c), a / t};
    double next = 0.0;
    for (const double x : at) {
      if (!(x >= 0.0)) continue;
      const double q = std::min(x, end), poly = b * q + c * q * q;
      if (!(std::fabs(poly) < 31.0)) return false;
      next = std::max(next, std::fabs(std::sqrt(q) * (a + poly)));
    }
    if (!(next <= 4.0)) return false;
    top = next * SLACK;
  }
  return true;
}

template <int MODE>
void launch_product(const NsParams &p, int form, int flip, hipStream_t st) {
  const int t = form == FORM_128 ? 128 : form == FORM_64 ? 64 : 32;
  // what the next product reads: whole tiles of its own
  int ti = form == FORM_SMALL ? (p.r + 31) / 32 : p.rp / t;
  const long long tj = (p.n + t - 1) / t, cus = vitk::cu_count();
  long long total = p.batch * (MODE <= POLY ? (long long)ti * (ti + 1) / 2 : ti * tj);
  if constexpr (MODE <= POLY) {
    // (two of 100 x 6500, 6 tiles: 317 -> 199 us; three of 128 x 3000, 9 tiles: 197 -> 131; nine of 70 x 2225, 27: 184 -> 204)
    if (form != FORM_SMALL && 16 * total <= cus) {
      form = FORM_SMALL;
      ti = p.rp / 32;
      total = p.batch * (long long)ti * (ti + 1) / 2;
    }
    // (1000 x 257, 45 tiles of 32: 129 -> 98 us; five of 192 x 192, 105: 98 -> 90; eight of 172 x 214, 168: 114 -> 125)
    if (form == FORM_SMALL && 2 * total <= cus) {
      const unsigned wgs = (unsigned)(p.batch * ti * (2 * ti + 1));  // twice the tiles a side
      if (MODE == GRAM && p.n > 512)
        hipLaunchKernelGGL((ns_lower_kernel<GRAM, 8>), dim3(wgs), dim3(512), 0, st, p, flip, 2 * ti);
      else
        hipLaunchKernelGGL((ns_lower_kernel<MODE, 4>), dim3(wgs), dim3(256), 0, st, p, flip, 2 * ti);
      return;
    }
  }
  const dim3 grid((unsigned)((total + 7) / 8 * 8));
  if (form == FORM_128)
    hipLaunchKernelGGL((ns_tile_kernel<MODE, 128, 8>), grid, dim3(512), 0, st, p, flip, (int)total);
  else if (form == FORM_64)
    hipLaunchKernelGGL((ns_tile_kernel<MODE, 64, 4>), grid, dim3(256), 0, st, p, flip, (int)total);
  else if ((MODE == GRAM ? p.n : p.r) > (MODE >= APPLY ? 256 : 512))  // more than one batch of loads a wave with four
    hipLaunchKernelGGL((ns_small_kernel<MODE, 8>), dim3((unsigned)total), dim3(512), 0, st, p, flip, ti);
  else
    hipLaunchKernelGGL((ns_small_kernel<MODE, 4>), dim3((unsigned)total), dim3(256), 0, st, p, flip, ti);
}

std::atomic<unsigned long long> g_one_lds{0};

int run(const char *who, NsParams *p, float *workspace, size_t bytes, hipStream_t st) {
  int form;
  const size_t need = plan(p, nullptr, &form);
  const dim3 block(256);
  if (form == FORM_ONE) {
    const int tr = (p->r + 31) / 32, tn = (p->n + 31) / 32;
    VITK_REQUIRE(vitk::fits_one_launch(p->batch, 64 * ONE_WAVES), "%s: too many matrices for one launch", who);
    const size_t lds = (size_t)tr * 32 * (one_pitch(tn) + one_pitch(tr)) * 16;
    if (vitk::reserve_lds(who, reinterpret_cast<const void *>(ns_one_kernel), 2 * ONE * one_pitch(ONE / 32) * 16, &g_one_lds))
      return 1;
    hipLaunchKernelGGL(ns_one_kernel, dim3(p->batch), dim3(64 * ONE_WAVES), lds, st, *p);
    return vitk::check_launch(who);
  }
  VITK_REQUIRE(workspace && bytes >= need, "%s: workspace of %zu bytes needed, %zu given", who, need,
               workspace ? bytes : 0);
  VITK_REQUIRE(vitk::aligned16(workspace), "%s: workspace is not 16-byte aligned", who);
  plan(p, workspace, &form);
  const long long yb = (long long)p->batch * (p->rp / 64) * (p->np / 64);
  VITK_REQUIRE(vitk::fits_one_launch(yb + 8, 256) && vitk::fits_one_launch(p->batch * (long long)PARTS, 256),
               "%s: too many matrices for one launch", who);
  hipLaunchKernelGGL(ns_norm_kernel, dim3(p->batch * PARTS), block, 0, st, *p);
  hipLaunchKernelGGL(ns_start_kernel, dim3((unsigned)yb), block, 0, st, *p, p->steps == 0 ? 1 : 0);
  for (int s = 0; s < p->steps; ++s) {
    launch_product<GRAM>(*p, form, s & 1, st);
    launch_product<POLY>(*p, form, s & 1, st);
    if (s + 1 < p->steps)
      launch_product<APPLY>(*p, form, s & 1, st);
    else
      launch_product<LAST>(*p, form, s & 1, st);
  }
  return vitk::check_launch(who);
}

size_t bytes_of(int32_t rows, int32_t cols, int32_t batch) {
  if (!size_ok(rows, cols, batch) || rows == 0 || cols == 0 || batch == 0) return 0;
  NsParams p = {};
  p.rows = rows, p.cols = cols, p.batch = batch;
  int form;
  return plan(&p, nullptr, &form);
}

int check(const char *who, int64_t rows, int64_t cols, int64_t batch, int steps, float a, float b, float c, float eps) {
  VITK_REQUIRE(size_ok(rows, cols, batch), "%s: bad shape", who);
  VITK_REQUIRE(steps >= 0 && steps <= 32, "%s: %d steps outside [0, 32]", who, steps);
  VITK_REQUIRE(eps >= 0.f && std::isfinite(eps), "%s: eps has to be a finite number >= 0", who);
  VITK_REQUIRE(bounded(a, b, c, steps), "%s: coefficients (%g, %g, %g) do not keep singular values bounded", who, a, b, c);
  return 0;
}

}  // namespace

extern "C" size_t vitk_newton_schulz_workspace_bytes(int32_t rows, int32_t cols, int32_t batch) {
  return bytes_of(rows, cols, batch);
}
extern "C" size_t vitk_muon_workspace_bytes(int32_t rows, int32_t cols, int32_t batch) {
  return bytes_of(rows, cols, batch);
}

extern "C" int vitk_newton_schulz_f32(const vitk_newton_schulz_args *a, vitk_stream_t stream) {
  const char *who = "vitk_newton_schulz_f32";
  VITK_REQUIRE(a != nullptr, "%s: null arguments", who);
  if (check(who, a->rows, a->cols, a->batch, a->steps, a->a, a->b, a->c, a->eps)) return 1;
  if (a->rows == 0 || a->cols == 0 || a->batch == 0) return 0;
  VITK_REQUIRE(a->x && a->out, "%s: null pointer", who);
  VITK_REQUIRE(a->ld_x >= a->cols && a->ld_out >= a->cols, "%s: row pitch below the columns", who);
  VITK_REQUIRE(a->batch == 1 || (a->stride_x >= 0 && a->stride_out >= (a->rows - 1) * a->ld_out + a->cols),
               "%s: matrices overlap", who);
  VITK_REQUIRE(a->x != a->out || ((a->rows == 1 || a->ld_x == a->ld_out) && (a->batch == 1 || a->stride_x == a->stride_out)),
               "%s: in place, x and out have to have one layout", who);
  NsParams p = {};
  p.x = a->x, p.out = a->out;
  p.ld_x = a->ld_x, p.stride_x = a->stride_x, p.ld_out = a->ld_out, p.stride_out = a->stride_out;
  p.rows = a->rows, p.cols = a->cols, p.batch = a->batch, p.steps = a->steps;
  p.flat = (a->ld_x == a->cols || a->rows == 1) && vitk::aligned16(a->x) && (a->batch == 1 || a->stride_x % 4 == 0);
  p.vec = vitk::aligned16(a->out) && a->ld_out % 4 == 0 && (a->batch == 1 || a->stride_out % 4 == 0);
  p.a = a->a, p.b = a->b, p.c = a->c, p.eps = a->eps;
  return run(who, &p, a->workspace, a->workspace_bytes, vitk::as_stream(stream));
}

extern "C" int vitk_muon_f32(const vitk_muon_args *a, vitk_stream_t stream) {
  const char *who = "vitk_muon_f32";
  VITK_REQUIRE(a != nullptr, "%s: null arguments", who);
  if (check(who, a->rows, a->cols, a->batch, a->steps, a->a, a->b, a->c, a->eps)) return 1;
  if (a->rows == 0 || a->cols == 0 || a->batch == 0) return 0;
  VITK_REQUIRE(a->p && a->g && a->m, "%s: null pointer", who);
  VITK_REQUIRE(a->p != a->m && a->p != a->g && a->m != a->g, "%s: p, g and m have to be different buffers", who);
  VITK_REQUIRE(a->ld >= a->cols, "%s: row pitch below the columns", who);
  VITK_REQUIRE(a->batch == 1 || a->stride >= (a->rows - 1) * a->ld + a->cols, "%s: matrices overlap", who);
  NsParams p = {};
  p.x = a->g, p.m = a->m, p.p = a->p;
  p.ld_x = p.ld_out = a->ld, p.stride_x = p.stride_out = a->stride;
  p.rows = a->rows, p.cols = a->cols, p.batch = a->batch, p.steps = a->steps;
  p.flat = (a->ld == a->cols || a->rows == 1) && vitk::aligned16(a->g) && vitk::aligned16(a->m) &&
           (a->batch == 1 || a->stride % 4 == 0);
  p.vec = vitk::aligned16(a->p) && a->ld % 4 == 0 && (a->batch == 1 || a->stride % 4 == 0);
  p.momentum = a->momentum, p.grad_scale = a->grad_scale, p.nesterov = a->nesterov;
  p.keep = 1.f - a->lr * a->weight_decay, p.step = a->lr * a->update_scale;
  p.a = a->a, p.b = a->b, p.c = a->c, p.eps = a->eps;
  return run(who, &p, a->workspace, a->workspace_bytes, vitk::as_stream(stream));
}
