// Shared by the forward and the backward of cross attention (cross_attention.hip, cross_attention_bwd.hip).
#pragma once
#include "common.h"

#include <algorithm>

namespace vitk {
namespace cross {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
  float *delta;  // backward: [B*H][Nq] dout . out / l
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
// The batch entry whose workgroups come `place`-th: the longest first, so that the last ones to start are short
// (only an order of work: every entry has one place).  Up to 64 entries, a lane each.
__device__ __forceinline__ int by_length(const Params &p, int place) {
  if (!p.len || p.B > 64) return place;
  const int lane = threadIdx.x & 63;
  const int mine = lane < p.B ? valid_keys(p, lane) : -1;
  int rank = 0;
  for (int j = 0; j < p.B; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    rank += other > mine || (other == mine && j < lane);
  }
  return __builtin_ctzll(__ballot(lane < p.B && rank == place));
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
// p0 p0', p0 p1', p1 p0', p0 p2', p2 p0', p1 p1' (p1 is at most 2^-8 of x and p2 2^-16, so the others are
// at most 2^-23 of x x' together, and mostly far less), summed in fp32 by
// v_mfma_f32_16x16x32_bf16: 16 times the rate of the fp32 instruction, so 2.7 times with six.  16 rows a wave
// instead of 32 halve what a wave keeps in registers (its own operand and its sums), and with four
// waves a SIMD instead of one or two the matrix cores work while other waves split and exponentiate.
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
__device__ __forceinline__ f32x4 product6(const Split8 &a, const Split8 &b, f32x4 acc) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[2], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[2], b.p[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[0], acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 all4(float x) { return f32x4{x, x, x, x}; }
__device__ __forceinline__ f32x4 zero4() { return all4(0.f); }

// Lane (c = lane & 15, g = lane >> 4) of the instruction supplies A[i = c][k = 8 g ..] and B[k = 8 g ..][j = c] and
// receives D[i = 4 g + r][j = c] in register r.  Two results for rows 0..15 and 16..31 are the operand
// B of a contraction over those 32 rows if slot (g, e) stands for row 4 g + e, e < 4, and 16 + 4 g + e - 4:
// the other operand is read in that order (Tile::columns).
// A tile of rows x DH in LDS: per row three parts of DH bf16, in units of 16 bytes.  Unit u of a part sits at
// u ^ spread(row), so that what is accessed together lies on different banks (64 of 4 bytes).  16 bytes a lane:
// lanes 0-3, 12-15, 20-27 go together, then the other 16 of 32, so a read along the columns takes unit u of
// rows 0-3 and 12-15 with unit u ^ 1 of rows 4-11.  A transposed read: eight rows of two neighbouring units.
template <int DH>
struct Tile {
  static constexpr int PART = DH / 8, ROW = 3 * PART;  // units
  __device__ static __forceinline__ int spread(int row) {
    const int high = (row >> 2) & 1;
    if constexpr (DH == 64) return (((row >> 1) & 3) << 1) | high;
    if constexpr (DH == 128) return ((row & 7) << 1) | high;
    return 3 * high;
  }
  __device__ static __forceinline__ void put(bf16x8 *tile, int row, int unit, const Split8 &x) {
#pragma unroll
    for (int k = 0; k < 3; ++k) tile[row * ROW + k * PART + (unit ^ spread(row))] = x.p[k];
  }
  // columns 32 step + 8 g .. + 7 of row `row` (= first + c)
  __device__ static __forceinline__ Split8 rows(const bf16x8 *tile, int row, int step, int g) {
    Split8 r;
#pragma unroll
    for (int k = 0; k < 3; ++k) r.p[k] = tile[row * ROW + k * PART + ((4 * step + g) ^ spread(row))];
    return r;
  }
  // column 16 block + c of rows first + 4 g .. + 3 and first + 16 + 4 g .. + 3
  __device__ static __forceinline__ Split8 columns(const bf16x8 *tile, int first, int block, int lane) {
    Split8 r;
    const int row = first + 4 * (lane >> 4) + ((lane & 15) >> 2), unit = 2 * block + ((lane & 3) >> 1);
    const __bf16 *base = reinterpret_cast<const __bf16 *>(tile) + 4 * (lane & 1);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const bf16x4 x = transposed(base + (row * ROW + k * PART + (unit ^ spread(row))) * 8);
      const bf16x4 y = transposed(base + ((row + 16) * ROW + k * PART + (unit ^ spread(row + 16))) * 8);
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
// two results (rows 0..15 and 16..31) as an operand
__device__ __forceinline__ Split8 split_pair(const f32x4 (&x)[2]) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = x[0][e], v[4 + e] = x[1][e];
  return split8(v);
}
// s += rows first .. first + 31 of a tile times this lane's row f (DH / 32 steps)
template <int DH>
__device__ __forceinline__ void rows_times(const bf16x8 *tile, int first, int c, int g, const Split8 (&f)[DH / 32],
                                           f32x4 (&s)[2]) {
#pragma unroll
  for (int i = 0; i < DH / 32; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) s[h] = product6(Tile<DH>::rows(tile, first + 16 * h + c, i, g), f[i], s[h]);
}
// acc^T[d][col] += tile^T[d][r] x[r][col], r in first .. first + 31
template <int DH>
__device__ __forceinline__ void add_columns(f32x4 (&acc)[DH / 16], const bf16x8 *tile, int first, int lane, const Split8 &x) {
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) acc[n] = product6(Tile<DH>::columns(tile, first, n, lane), x, acc[n]);
}
// over the four lanes that hold one column: exchanging the upper half of one copy with the lower half of another
// leaves {own, other} in the two; then the same with neighbouring rows of 16 lanes.  (Written out: of the
// builtin's two results this compiler keeps one.  The wait is the one it puts before the exchange.)
__device__ __forceinline__ float column_max(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = y = fmaxf(x, y);
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// this lane's part of a row (columns 32 i + 8 g ..), which has to be there; every load in flight at once (a branch
// around each, as for columns behind dh, would wait for one after the other)
template <int DH>
__device__ __forceinline__ void load_raw(float (&x)[DH / 32][8], const float *row, int g, const Params &p) {
  if (p.vec) {
#pragma unroll
    for (int i = 0; i < DH / 32; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 32 * i + 8 * g + 4 * h;
        const f32x4 v = *reinterpret_cast<const f32x4 *>(row + (d < p.dh ? d : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][4 * h + e] = v[e];
      }
  } else {
#pragma unroll
    for (int i = 0; i < DH / 32; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = row[min(32 * i + 8 * g + e, p.dh - 1)];
  }
#pragma unroll
  for (int i = 0; i < DH / 32; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (32 * i + 8 * g + e >= p.dh) x[i][e] = 0.f;
}
// that times `scale`, split; zeros for a row that is not there
template <int DH>
__device__ __forceinline__ void split_row(Split8 (&f)[DH / 32], float (&x)[DH / 32][8], bool ok, float scale) {
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = ok ? x[i][e] * scale : 0.f;
    f[i] = split8(x[i]);
  }
}
// column c of acc^T to a row
template <int DH>
__device__ __forceinline__ void store_row(float *row, const f32x4 (&acc)[DH / 16], float f, int g, int dh, bool vec) {
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = acc[n][e] * f;
    store_quad(row, 16 * n + 4 * g, dh, vec, x);
  }
}

// NW waves, GROUPS of 16 rows (or keys); OTHER = waves that share a group and deal the 32-row tiles of a stage of
// the other side.  A stage (two tensors) is loaded into registers, split and put into one of two buffers while
// the waves work on the other one: half of the waves before their products, half after them, so that on each
// SIMD one wave splits while the other multiplies.  (With OTHER = 2 a stage is twice as long and has one buffer:
// two would leave room for one workgroup a CU.  So have four waves of OTHER = 1, for more workgroups a CU.)
template <int DH, int NW, int GROUPS>
struct Shape {
  static constexpr int OTHER = NW / GROUPS, STAGE = 32 * OTHER, BUFFERS = OTHER == 1 && NW == 8 ? 2 : 1;
  static constexpr int THREADS = 64 * NW, HALF = STAGE * DH / 8, TASKS = (2 * HALF + THREADS - 1) / THREADS;
  static constexpr int UNITS = STAGE * Tile<DH>::ROW;  // of a tensor; a buffer holds two
};
// Eight columns of a row per task: first those of x, then those of y.
template <int DH, int NW, int GROUPS>
struct Stage {
  typedef Shape<DH, NW, GROUPS> S;
  float v[S::TASKS][8];
  __device__ static __forceinline__ int task(int u) { return threadIdx.x + S::THREADS * u; }
  __device__ static __forceinline__ bool any(int u) { return 2 * S::HALF % S::THREADS == 0 || task(u) < 2 * S::HALF; }
  __device__ static __forceinline__ bool is_y(int u) { return task(u) >= S::HALF; }
  __device__ static __forceinline__ int row(int u) { return (task(u) - (is_y(u) ? S::HALF : 0)) / (DH / 8); }
  __device__ static __forceinline__ int unit(int u) { return task(u) % (DH / 8); }
  // at(y, row): the row's first element.  Every load is issued, its place clamped (see load_raw); `clean` before
  // the values are used.
  template <class At>
  __device__ __forceinline__ void fetch(const Params &p, int first, int end, At at) {
    if (first >= end) {
#pragma unroll
      for (int u = 0; u < S::TASKS; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
      return;
    }
    if (p.vec) {
#pragma unroll
      for (int u = 0; u < S::TASKS; ++u) {
        int r = row(u), d0 = unit(u) * 8;
        if constexpr (DH == 96) asm volatile("" : "+v"(r), "+v"(d0));  // (no place to keep what follows from them)
        const float *from = at(is_y(u), min(first + r, end - 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = d0 + 4 * h;
          const f32x4 x = *reinterpret_cast<const f32x4 *>(from + (d < p.dh ? d : 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][4 * h + e] = x[e];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < S::TASKS; ++u) {
        const float *from = at(is_y(u), min(first + row(u), end - 1));
        int d = unit(u) * 8;
        asm volatile("" : "+v"(d));  // (the compiler would keep eight places a task in registers for the whole loop)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[u][e] = from[min(d + e, p.dh - 1)];
      }
    }
  }
  // what was fetched: zeros for rows behind the end and columns behind dh
  __device__ __forceinline__ void clean(const Params &p, int first, int end) {
    if (first + S::STAGE <= end && p.dh == DH) return;
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u) {
      int r = row(u), d0 = unit(u) * 8;
      if constexpr (DH == 96) asm volatile("" : "+v"(r), "+v"(d0));
      const int columns = first + r < end ? p.dh - d0 : 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e >= columns) v[u][e] = 0.f;
    }
  }
  __device__ __forceinline__ void put(bf16x8 *buffer) const {
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u)
      if (any(u)) Tile<DH>::put(buffer + (is_y(u) ? S::UNITS : 0), row(u), unit(u), split8(v[u]));
  }
};

// Groups of 16 rows (or keys) in a workgroup, and its waves.  Eight groups split the other side's tiles for 128
// rows at once.  Four groups are four waves, of which several workgroups are on a CU, if there are at least as
// many such workgroups as CUs; otherwise eight, so that two share a group's other side (64 columns, forward, eight
// waves -> four: 64 x 64, 2048 heads: 40 -> 33 us; 50 x 900, 24 heads: 18 -> 23).  More than 64 rows are cut into
// blocks of 64 where the last block of 128 were half empty and that is a sixth of the rows or more (147 x 197, 320
// heads: forward 42 -> 33, row gradient 19 less; 300 x 500 x 96, 96 heads: 72 -> 48 and 50 less; 150 x 1000 x 128:
// 91 -> 102), up to `half` on the other side, and up to `any` on the other side always (row gradient of 512 x 128,
// 192 heads: 5 less; 512 x 197: 2 more; key gradients of 16 rows x 1000, 128 heads of 96: 7 less).
struct Block {
  int groups, waves;
};
inline Block plan_block(long long own, long long other, long long heads, bool small, int half, int any) {
  if (own <= 32) return {2, 4};
  const long long blocks = (own + 63) / 64;
  small = small && heads * blocks >= vitk::cu_count();
  if (own <= 64) return {4, small ? 4 : 8};
  const bool halves = blocks % 2 == 1 && blocks <= 5;
  return small && ((halves && other <= half) || other <= any) ? Block{4, 4} : Block{8, 8};
}
// Over how many workgroups the other side of a block is split: the least of whole rounds over the device's
// places for workgroups (a last round that is hardly filled costs as much as a full one) plus writing and
// adding the parts.  `us`: time of a whole block by its products; `stage_us`: of the loads, products and barriers of 64
// on the other side, one after the other; `part_us`: of one part of the results.  (10 x 814 x 64, 42 heads: forward
// 25 us in three parts, 13 in thirteen.)
inline int plan_splits(long long wgs, long long places, long long stages, double us, double stage_us, double part_us) {
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 16 && (s == 1 || s <= stages); ++s) {
    const double block = std::max(us / s, (double)((stages + s - 1) / s) * stage_us);
    const double t = (double)((wgs * s + places - 1) / places) * block + (s > 1 ? 5.0 + s * part_us : 0.0);
    if (s == 1 || t < least) best = s, least = t;
  }
  return best;
}

// Query rows of a key head and keys that the kernels' row numbers (and what they add to them) hold.
inline bool few_enough_rows(const vitk_cross_sdpa_args *a) {
  return (long long)(a->H / a->Hkv) * a->Nq < 2147482624 && a->Nk < 2147482624;
}

// Argument checks both directions share; fills everything but the launch plan.
int check_args(const char *who, const vitk_cross_sdpa_args *a, bool backward, Params *p);

}  // namespace cross
}  // namespace vitk
