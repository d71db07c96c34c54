// Shared by the forward and the backward of cross attention (cross_attention.hip, cross_attention_bwd.hip).
#pragma once
#include "common.h"

namespace vitk {
namespace cross {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

// One operand: element (b, n, h, d) at ptr[(b*N + n)*ld + h*dh + d].
struct Operand {
  const float *ptr;
  long long ld;
};
struct Result {
  float *ptr;
  long long ld;
};

struct Params {
  Operand q, k, v, o, dout;
  Result out, dq, dk, dv;
  const int32_t *len;
  float *stats;  // [B*H][Nq][2]
  float *delta;  // backward: [B*H][Nq] dout . out
  // forward, keys split: [splits][B*H][Nq][dh] unnormalised sums, then [splits][B*H][Nq][2];
  // backward, keys or rows split: [splits][B][N][heads][dh] of one gradient (of dk, then of dv)
  float *part;
  int B, H, Hkv, G, Nq, Nk, dh;
  int rows;      // G * Nq: the query rows that share one key head, head by head
  int blocks;    // row (or key) blocks per (batch, key head)
  int splits, chunk;
  float scale, c;  // c = scale * log2(e): softmax in powers of two
  bool vec;        // 16-byte aligned operands, ld and dh multiples of 4
};

// Row r of key head hk: query head hk*G + r/Nq, token r%Nq.
__device__ __forceinline__ long long row_offset(const Params &p, long long ld, int b, int hk, int r) {
  const int j = r / p.Nq, n = r - j * p.Nq;
  return ((long long)b * p.Nq + n) * ld + (long long)(hk * p.G + j) * p.dh;
}
__device__ __forceinline__ long long row_stat(const Params &p, int b, int hk, int r) {  // [B*H][Nq] index
  return ((long long)b * p.H + (long long)hk * p.G) * p.Nq + r;
}
__device__ __forceinline__ long long key_offset(const Params &p, long long ld, int b, int hk, int n) {
  return ((long long)b * p.Nk + n) * ld + (long long)hk * p.dh;
}
__device__ __forceinline__ int valid_keys(const Params &p, int b) {
  return p.len ? min(max(p.len[b], 0), p.Nk) : p.Nk;
}

// Columns d .. d+3 of a row; zeros behind dh.
__device__ __forceinline__ f32x4 load_quad(const float *row, int d, int dh, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec) {
    if (d < dh) r = *reinterpret_cast<const f32x4 *>(row + d);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < dh) r[e] = row[d + e];
  }
  return r;
}
__device__ __forceinline__ void store_quad(float *row, int d, int dh, bool vec, f32x4 x) {
  if (vec) {
    if (d < dh) *reinterpret_cast<f32x4 *>(row + d) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < dh) row[d + e] = x[e];
  }
}

// ------------------------------------------------------------------ fp32 products in three parts
// x = p0 + p1 + p2 exactly: each part the bf16 nearest to what is left (8 + 8 + 8 bits and two signs
// cover the 24 of fp32).  A product of two such numbers to fp32 accuracy is the six part products
// p0 p0', p0 p1', p1 p0', p0 p2', p2 p0', p1 p1' (the others are below 2^-26), summed in fp32 by
// v_mfma_f32_32x32x16_bf16: 16 times the rate of the fp32 instruction, so 2.7 times with six.
struct Split8 {
  bf16x8 p[3];
};
__device__ __forceinline__ void split2(f32x2 x, bf16x2 (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    part[k] = __builtin_convertvector(x, bf16x2);
    if (k < 2) {
      x[0] -= (float)part[k][0];
      x[1] -= (float)part[k][1];
    }
  }
}
__device__ __forceinline__ Split8 split8(const float (&x)[8]) {
  Split8 r;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    bf16x2 part[3];
    split2(f32x2{x[e], x[e + 1]}, part);
#pragma unroll
    for (int k = 0; k < 3; ++k) r.p[k][e] = part[k][0], r.p[k][e + 1] = part[k][1];
  }
  return r;
}
// acc += a b, the small products first
__device__ __forceinline__ f32x16 product6(const Split8 &a, const Split8 &b, f32x16 acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// A tile of rows x DH in LDS: per row three parts of DH bf16, in units of 16 bytes.  Unit u of a part sits at
// u ^ spread(row), which puts 16 rows of one unit (a read along the columns) and four rows of four
// neighbouring units (a transposed read) on different banks.
template <int DH>
struct Tile {
  static constexpr int PART = DH / 8, ROW = 3 * PART;  // units
  __device__ static __forceinline__ int spread(int row) {
    if constexpr (DH == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    if constexpr (DH == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    return (row >> 2) & 3;
  }
  __device__ static __forceinline__ void put(bf16x8 *tile, int row, int unit, const Split8 &x) {
#pragma unroll
    for (int k = 0; k < 3; ++k) tile[row * ROW + k * PART + (unit ^ spread(row))] = x.p[k];
  }
  // operand of 16 columns: lane (c, g) takes columns 16 step + 8 g .. + 7 of row `row` (= first + c)
  __device__ static __forceinline__ Split8 rows(const bf16x8 *tile, int row, int step, int g) {
    Split8 r;
#pragma unroll
    for (int k = 0; k < 3; ++k) r.p[k] = tile[row * ROW + k * PART + ((2 * step + g) ^ spread(row))];
    return r;
  }
  // operand of 16 rows of the transposed tile: lane (c, g) takes column 32 block + c of rows
  // first + 4 g .. + 3 and first + 8 + 4 g .. + 3, the rows whose products registers 8 s .. 8 s + 7 of a
  // 32 x 32 result hold (first = 16 s)
  __device__ static __forceinline__ Split8 columns(const bf16x8 *tile, int first, int block, int lane) {
    Split8 r;
    const int row = first + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int unit = 4 * block + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const __bf16 *base = reinterpret_cast<const __bf16 *>(tile) + 4 * (lane & 1);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const bf16x4 x = transposed(base + (row * ROW + k * PART + (unit ^ spread(row))) * 8);
      const bf16x4 y = transposed(base + ((row + 8) * ROW + k * PART + (unit ^ spread(row + 8))) * 8);
      r.p[k] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return r;
  }
  // lane l of each 16 gets rows 0..3 of column l of the 4 x 16 block whose row l / 4, columns 4 (l % 4) .. + 3,
  // its address names
  __device__ static __forceinline__ bf16x4 transposed(const __bf16 *at) {
    const i16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)(at));
    return __builtin_bit_cast(bf16x4, r);
  }
};
// registers 8 s .. 8 s + 7 of a 32 x 32 result as an operand
__device__ __forceinline__ Split8 split_half(const f32x16 &x, int s) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[8 * s + e];
  return split8(v);
}
// columns d .. d + 7 of a row; zeros behind dh
__device__ __forceinline__ void load_eight(const float *row, int d, const Params &p, float (&x)[8]) {
  const f32x4 a = load_quad(row, d, p.dh, p.vec), b = load_quad(row, d + 4, p.dh, p.vec);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
}

// Argument checks both directions share; fills everything but the launch plan.
int check_args(const char *who, const vitk_cross_sdpa_args *a, bool backward, Params *p);

}  // namespace cross
}  // namespace vitk
