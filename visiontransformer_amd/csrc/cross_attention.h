// Shared by the forward and the backward of cross attention (cross_attention.hip, cross_attention_bwd.hip).
#pragma once
#include "common.h"

namespace vitk {
namespace cross {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

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
  float *part;   // forward, keys split: [splits][B*H][Nq][dh] unnormalised sums, then [splits][B*H][Nq][2]
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

// Argument checks both directions share; fills everything but the launch plan.
int check_args(const char *who, const vitk_cross_sdpa_args *a, bool backward, Params *p);

}  // namespace cross
}  // namespace vitk
