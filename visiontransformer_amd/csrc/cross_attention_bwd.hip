// Cross attention backward without atomics:
//   dQ (and delta[row] = dout . out / l): one workgroup per block of rows, all keys in order;
//   dK, dV: one workgroup per block of keys of one (batch, key head), all rows that read them in order.
// Both rebuild the probabilities from the stored row statistics,
//   e = exp2(c s - m),  p = e / l,  ds = p (dout v^T - delta),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T dout,
// with dout / l and delta / l in the place of dout and delta, so that e needs no factor, and with -m and
// -delta / l as what the products are added to;
// the products are fp32 in three bf16 parts, arranged as in the forward: the accumulator of the first
// product is the operand of the next.  That is seven products where five would do (s and dp are formed
// twice); one pass would have to add dQ (or dK and dV) up across workgroups.
// Blocks of up to 128 rows (keys), 16 a wave; with fewer, two waves may share a group and deal the tiles of the
// other side.  Where the blocks are too few for the device, the other side is split over workgroups and
// the parts are added in order by a second launch.
// Bound by the matrix cores (512 x 1536 x 96, 128 heads of which 4 share a key head: dQ 328 us, dK and dV 437, 1060
// TFLOP/s of bf16 products each); few keys by the start and the end of a workgroup.
#include "cross_attention.h"

#include <algorithm>

namespace {

using namespace vitk::cross;

// The other wave's sums of the same rows (keys) are added through LDS.
template <int NB>
__device__ __forceinline__ void give(float *box, const f32x4 (&acc)[NB]) {
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) box[(4 * n + e) * 64] = acc[n][e];
}
template <int NB>
__device__ __forceinline__ void take(const float *box, f32x4 (&acc)[NB]) {
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] += box[(4 * n + e) * 64];
}

// Workgroups of four waves that a CU holds, with one group of rows (or keys: 2) a wave.  (Of 128 columns one,
// which is slower than eight waves that share the groups: 64 x 64, 2048 heads, both together 370 -> 386 us.)
constexpr int dq_resident(int dh) { return dh <= 32 ? 4 : dh <= 64 ? 3 : 2; }

template <int DH, int NW, int RW>
__global__ __launch_bounds__(64 * NW, NW == 4 && RW == 4 ? dq_resident(DH) : NW == 8 || DH <= 64 ? 2 : 1)
void cross_dq_kernel(const Params p) {
  typedef Shape<DH, NW, RW> S;
  constexpr int JOIN = S::OTHER > 1 ? RW * 64 * (DH / 4) * 4 : 0;
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BUFFERS * S::UNITS * 16 > JOIN ? 2 * S::BUFFERS * S::UNITS * 16 : JOIN];
  bf16x8 *buffers = reinterpret_cast<bf16x8 *>(lds);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RW, kg = wave / RW;
  long long wg = blockIdx.x;
  const int rb = (int)(wg % p.blocks);
  wg /= p.blocks;
  const int hk = (int)(wg % p.Hkv);
  wg /= p.Hkv;
  const int split = (int)(wg % p.splits), b = by_length(p, (int)(wg / p.splits));
  const int len = valid_keys(p, b), row = (rb * RW + rg) * 16 + c;
  const int k0 = min((long long)split * p.chunk, (long long)len), k1 = min((long long)k0 + p.chunk, (long long)len);
  const bool row_ok = row < p.rows;
  Split8 q[DH / 32], dout[DH / 32];  // q times scale log2(e); dout / l
  float m = 0.f, delta = 0.f;        // delta / l
  {
    const int r = row_ok ? row : 0;
    float f = 0.f;
    const long long st = row_stat(p, b, hk, r);
    if (row_ok) {
      m = p.stats[2 * st];
      const float l = p.stats[2 * st + 1];
      f = l == 0.f ? 0.f : 1.f / l;
    }
    float x[DH / 32][8], y[DH / 32][8], z[DH / 32][8];
    load_raw<DH>(x, p.q.ptr + row_offset(p, p.q.ld, b, hk, r), g, p);
    load_raw<DH>(y, p.dout.ptr + row_offset(p, p.dout.ld, b, hk, r), g, p);
    load_raw<DH>(z, p.o.ptr + row_offset(p, p.o.ld, b, hk, r), g, p);
    split_row<DH>(q, x, row_ok, p.c);
#pragma unroll
    for (int i = 0; i < DH / 32; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += row_ok ? y[i][e] * z[i][e] : 0.f;
    split_row<DH>(dout, y, row_ok, f);
    delta = column_sum(delta) * f;
    if (row_ok && g == 0 && kg == 0 && split == 0) p.delta[st] = delta;
  }
  f32x4 dq[DH / 16];
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) dq[n] = zero4();
  Stage<DH, NW, RW> next;
  auto at = [&](bool y, int n) {
    return y ? p.v.ptr + key_offset(p, p.v.ld, b, hk, n) : p.k.ptr + key_offset(p, p.k.ld, b, hk, n);
  };
  const bool early = wave < NW / 2, empty = (rb * RW + rg) * 16 >= p.rows;
  next.fetch(p, k0, k1, at);
  if constexpr (S::BUFFERS == 2) {
    next.clean(p, k0, k1);
    next.put(buffers);
    next.fetch(p, k0 + S::STAGE, k1, at);
    __syncthreads();
  }
  for (int t = k0, n = 0; t < k1; t += S::STAGE, n ^= S::BUFFERS - 1) {
    const bf16x8 *kt = buffers + n * 2 * S::UNITS, *vt = kt + S::UNITS;
    auto advance = [&] {
      next.clean(p, t + (S::BUFFERS - 1) * S::STAGE, k1);
      next.put(buffers + (S::BUFFERS - 1 - n) * 2 * S::UNITS);
      if constexpr (S::BUFFERS == 1) __syncthreads();
      next.fetch(p, t + S::BUFFERS * S::STAGE, k1, at);
    };
    if (S::BUFFERS == 1 || early) advance();
    const int first = 32 * kg;
    if (!empty && t + first < k1) {
      f32x4 s[2] = {all4(-m), all4(-m)}, ds[2] = {all4(-delta), all4(-delta)};
      rows_times<DH>(kt, first, c, g, q, s);
      rows_times<DH>(vt, first, c, g, dout, ds);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) ds[h][e] *= __builtin_amdgcn_exp2f(s[h][e]);
      if (t + first + 32 > k1) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t + first + 16 * h + 4 * g + e >= k1) ds[h][e] = 0.f;
      }
      add_columns<DH>(dq, kt, first, lane, split_pair(ds));
    }
    if (S::BUFFERS == 2 && !early) advance();
    __syncthreads();
  }
  if constexpr (S::OTHER > 1) {
    float *box = reinterpret_cast<float *>(lds) + rg * 64 * (DH / 4) + lane;
    __syncthreads();
    if (kg == 1) give<DH / 16>(box, dq);
    __syncthreads();
    if (kg == 1) return;
    take<DH / 16>(box, dq);
  }
  if (!row_ok) return;
  if (p.splits > 1) {
    const long long pitch = (long long)p.H * p.dh, all = (long long)p.B * p.Nq * pitch;
    store_row<DH>(p.part + split * all + row_offset(p, pitch, b, hk, row), dq, p.scale, g, p.dh, p.dh % 4 == 0);
  } else {
    store_row<DH>(p.dq.ptr + row_offset(p, p.dq.ld, b, hk, row), dq, p.scale, g, p.dh, p.vec);
  }
}

template <int DH, int NW, int KG>
__global__ __launch_bounds__(64 * NW, 2)
void cross_dkv_kernel(const Params p) {
  typedef Shape<DH, NW, KG> S;
  constexpr int JOIN = S::OTHER > 1 ? KG * 64 * (DH / 2) * 4 : 0;
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BUFFERS * S::UNITS * 16 > JOIN ? 2 * S::BUFFERS * S::UNITS * 16 : JOIN];
  __shared__ __attribute__((aligned(16))) float rm[S::BUFFERS][S::STAGE], rd[S::BUFFERS][S::STAGE];
  bf16x8 *buffers = reinterpret_cast<bf16x8 *>(lds);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave % KG, rg = wave / KG;
  long long wg = blockIdx.x;
  const int kb = (int)(wg % p.blocks);
  wg /= p.blocks;
  const int hk = (int)(wg % p.Hkv);
  wg /= p.Hkv;
  const int split = (int)(wg % p.splits), b = by_length(p, (int)(wg / p.splits));
  const int len = valid_keys(p, b), key = (kb * KG + kg) * 16 + c;
  const bool key_ok = key < len;
  Split8 k[DH / 32], v[DH / 32];
  if (kb * KG * 16 < len) {
    float x[DH / 32][8], y[DH / 32][8];
    load_raw<DH>(x, p.k.ptr + key_offset(p, p.k.ld, b, hk, key_ok ? key : 0), g, p);
    load_raw<DH>(y, p.v.ptr + key_offset(p, p.v.ld, b, hk, key_ok ? key : 0), g, p);
    split_row<DH>(k, x, key_ok, p.c);
    split_row<DH>(v, y, key_ok, 1.f);
  }
  f32x4 dk[DH / 16], dv[DH / 16];
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) dk[n] = zero4(), dv[n] = zero4();
  // a block behind the length has nothing to add
  const int r0 = min((long long)split * p.chunk, (long long)p.rows);
  const int r1 = kb * KG * 16 < len ? (int)min((long long)r0 + p.chunk, (long long)p.rows) : r0;
  Stage<DH, NW, KG> next;
  auto at = [&](bool y, int r) {
    return y ? p.dout.ptr + row_offset(p, p.dout.ld, b, hk, r) : p.q.ptr + row_offset(p, p.q.ld, b, hk, r);
  };
  float sm = 0.f, sd = 0.f, sl[S::TASKS] = {};
  auto fetch = [&](int t) {
    next.fetch(p, t, r1, at);
    if (t >= r1) return;
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u)  // l of a task's row
      sl[u] = p.stats[2 * row_stat(p, b, hk, min(t + next.row(u), r1 - 1)) + 1];
    if (threadIdx.x < S::STAGE) {
      const long long st = row_stat(p, b, hk, min(t + (int)threadIdx.x, r1 - 1));
      sm = p.stats[2 * st], sd = p.delta[st];
    }
  };
  auto put = [&](int n, int t) {
    next.clean(p, t, r1);
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u) {  // dout / l
      const float f = !next.is_y(u) ? 1.f : sl[u] == 0.f ? 0.f : 1.f / sl[u];
#pragma unroll
      for (int e = 0; e < 8; ++e) next.v[u][e] *= f;
    }
    next.put(buffers + n * 2 * S::UNITS);
    if (threadIdx.x < S::STAGE) {  // a row that is not there: exp2(0) times zeros
      const bool there = t + (int)threadIdx.x < r1;
      rm[n][threadIdx.x] = there ? -sm : 0.f, rd[n][threadIdx.x] = there ? -sd : 0.f;
    }
  };
  const bool early = wave < NW / 2, empty = (kb * KG + kg) * 16 >= len;
  fetch(r0);
  if constexpr (S::BUFFERS == 2) {
    put(0, r0);
    fetch(r0 + S::STAGE);
    __syncthreads();
  }
  for (int t = r0, n = 0; t < r1; t += S::STAGE, n ^= S::BUFFERS - 1) {
    const bf16x8 *qt = buffers + n * 2 * S::UNITS, *gt = qt + S::UNITS;
    auto advance = [&] {
      put(S::BUFFERS - 1 - n, t + (S::BUFFERS - 1) * S::STAGE);
      if constexpr (S::BUFFERS == 1) __syncthreads();
      fetch(t + S::BUFFERS * S::STAGE);
    };
    if (S::BUFFERS == 1 || early) advance();
    const int first = 32 * rg;
    if (!empty && t + first < r1) {
      f32x4 s[2], ds[2];  // start from -m and -delta / l of their rows
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = *reinterpret_cast<const f32x4 *>(rm[n] + first + 16 * h + 4 * g);
        ds[h] = *reinterpret_cast<const f32x4 *>(rd[n] + first + 16 * h + 4 * g);
      }
      rows_times<DH>(qt, first, c, g, k, s);
      rows_times<DH>(gt, first, c, g, v, ds);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][e] = __builtin_amdgcn_exp2f(s[h][e]);
          ds[h][e] *= s[h][e];
        }
      add_columns<DH>(dv, gt, first, lane, split_pair(s));
      add_columns<DH>(dk, qt, first, lane, split_pair(ds));
    }
    if (S::BUFFERS == 2 && !early) advance();
    __syncthreads();
  }
  if constexpr (S::OTHER > 1) {
    float *box = reinterpret_cast<float *>(lds) + kg * 64 * (DH / 2) + lane;
    __syncthreads();
    if (rg == 1) give<DH / 16>(box, dk), give<DH / 16>(box + 64 * (DH / 4), dv);
    __syncthreads();
    if (rg == 1) return;
    take<DH / 16>(box, dk), take<DH / 16>(box + 64 * (DH / 4), dv);
  }
  if (key >= p.Nk) return;
  if (!key_ok) {  // (whatever its column held)
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) dk[n] = zero4(), dv[n] = zero4();
  }
  if (p.splits > 1) {
    const long long pitch = (long long)p.Hkv * p.dh, all = (long long)p.B * p.Nk * pitch;
    const long long at = key_offset(p, pitch, b, hk, key);
    store_row<DH>(p.part + split * all + at, dk, p.scale, g, p.dh, p.dh % 4 == 0);
    store_row<DH>(p.part + (p.splits + split) * all + at, dv, 1.f, g, p.dh, p.dh % 4 == 0);
  } else {
    store_row<DH>(p.dk.ptr + key_offset(p, p.dk.ld, b, hk, key), dk, p.scale, g, p.dh, p.vec);
    store_row<DH>(p.dv.ptr + key_offset(p, p.dv.ld, b, hk, key), dv, 1.f, g, p.dh, p.vec);
  }
}

// Few keys: all of a (batch, key head) in one workgroup of four waves, so dQ is complete here too: five products
// instead of seven, and each row is read once.  Each wave forms p and ds of its 16 keys with a stage of 32 rows
// and adds to dK and dV; ds goes through LDS as [key][row], and dQ^T[d][row] += K^T ds is dealt to the waves by
// blocks of 16 x 16.  K is there times scale log2(e), for the scores.  With fewer heads than places, rows are split.
// 147 x 50 x 64, 384 heads: 33 us, 50 x 50, 512 heads 18, 900 x 50, 24 heads, split, 24 (dQ, then dK and dV took 56,
// 28 and 43).  (64 columns fill the registers of two workgroups a CU.)
constexpr int FEW_KEYS = 64;
constexpr int short_resident(int dh) { return dh <= 32 ? 3 : 2; }
template <int DH>
__global__ __launch_bounds__(256, short_resident(DH)) void cross_short_kernel(const Params p) {
  typedef Shape<DH, 4, 4> S;
  typedef Tile<32> Turn;
  constexpr int UNITS = DH / 8;  // of a row of a stage: that many lanes load it
  static_assert(DH <= 64 && 64 % UNITS == 0, "the lanes of a row are neighbours in a wave");
  __shared__ __attribute__((aligned(16))) bf16x8 stage[2 * S::UNITS], kt[FEW_KEYS * Tile<DH>::ROW], turn[FEW_KEYS * Turn::ROW];
  __shared__ __attribute__((aligned(16))) float rm[32], rd[32];
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  long long wg = blockIdx.x;
  const int hk = (int)(wg % p.Hkv);
  wg /= p.Hkv;
  const int split = (int)(wg % p.splits), b = (int)(wg / p.splits);
  const int len = valid_keys(p, b), key = wave * 16 + c;
  const bool key_ok = key < len, empty = wave * 16 >= len;
  Split8 k[DH / 32], v[DH / 32];
  {
    float x[DH / 32][8] = {}, y[DH / 32][8] = {};
    if (len > 0) {
      load_raw<DH>(x, p.k.ptr + key_offset(p, p.k.ld, b, hk, key_ok ? key : 0), g, p);
      load_raw<DH>(y, p.v.ptr + key_offset(p, p.v.ld, b, hk, key_ok ? key : 0), g, p);
    }
    split_row<DH>(k, x, key_ok, p.c);
    split_row<DH>(v, y, key_ok, 1.f);
  }
  f32x4 dk[DH / 16], dv[DH / 16];
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) dk[n] = zero4(), dv[n] = zero4();
  const int r0 = min((long long)split * p.chunk, (long long)p.rows), r1 = min((long long)r0 + p.chunk, (long long)p.rows);
  Stage<DH, 4, 4> next;
  float o[S::TASKS][8] = {}, m[S::TASKS] = {}, l[S::TASKS] = {};  // of a task's row of dout
  auto at = [&](bool y, int r) {
    return y ? p.dout.ptr + row_offset(p, p.dout.ld, b, hk, r) : p.q.ptr + row_offset(p, p.q.ld, b, hk, r);
  };
  auto fetch = [&](int t) {
    next.fetch(p, t, r1, at);
    if (t >= r1) return;
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u) {
      if (!next.any(u) || !next.is_y(u)) continue;
      const int r = min(t + next.row(u), r1 - 1);
      const long long st = 2 * row_stat(p, b, hk, r);
      m[u] = p.stats[st], l[u] = p.stats[st + 1];
      const float *from = p.o.ptr + row_offset(p, p.o.ld, b, hk, r);
      int d = next.unit(u) * 8;
      if (p.vec) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(from + (d < p.dh ? d : 0)),
                    y = *reinterpret_cast<const f32x4 *>(from + (d + 4 < p.dh ? d + 4 : 0));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][e] = x[e], o[u][4 + e] = y[e];
      } else {
        asm volatile("" : "+v"(d));  // (as in Stage::fetch)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[u][e] = from[min(d + e, p.dh - 1)];
      }
    }
  };
  auto put = [&](int t) {
    next.clean(p, t, r1);
#pragma unroll
    for (int u = 0; u < S::TASKS; ++u) {
      if (!next.any(u) || !next.is_y(u)) continue;
      const bool there = t + next.row(u) < r1;  // if not: exp2(0) times zeros
      const float f = !there || l[u] == 0.f ? 0.f : 1.f / l[u];
      float delta = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        delta += there && next.unit(u) * 8 + e < p.dh ? next.v[u][e] * o[u][e] : 0.f;
        next.v[u][e] *= f;
      }
#pragma unroll
      for (int x = 1; x < UNITS; x *= 2) delta += __shfl_xor(delta, x, 64);
      if (next.unit(u) == 0) rm[next.row(u)] = there ? -m[u] : 0.f, rd[next.row(u)] = -(delta * f);
    }
    next.put(stage);
  };
  fetch(r0);
  bf16x4 *half = reinterpret_cast<bf16x4 *>(turn);
  auto turn_at = [&](int part, int h) {  // rows 16 h + 4 g .. + 3 of this lane's key
    return 2 * (key * Turn::ROW + part * Turn::PART + ((2 * h + (g >> 1)) ^ Turn::spread(key))) + (g & 1);
  };
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) Tile<DH>::put(kt, key, 4 * i + g, k[i]);
#pragma unroll
  for (int part = 0; part < 3; ++part)
#pragma unroll
    for (int h = 0; h < 2; ++h) half[turn_at(part, h)] = bf16x4{};  // keys that are not there
  const bf16x8 *qt = stage, *gt = stage + S::UNITS;
  for (int t = r0; t < r1; t += 32) {
    put(t);
    __syncthreads();
    fetch(t + 32);
    if (!empty) {
      f32x4 s[2], ds[2];  // start from -m and -delta / l of their rows
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = *reinterpret_cast<const f32x4 *>(rm + 16 * h + 4 * g);
        ds[h] = *reinterpret_cast<const f32x4 *>(rd + 16 * h + 4 * g);
      }
      rows_times<DH>(qt, 0, c, g, k, s);
      rows_times<DH>(gt, 0, c, g, v, ds);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][e] = __builtin_amdgcn_exp2f(s[h][e]);
          ds[h][e] = key_ok ? ds[h][e] * s[h][e] : 0.f;
        }
      const Split8 x = split_pair(ds);
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        half[turn_at(part, 0)] = __builtin_shufflevector(x.p[part], x.p[part], 0, 1, 2, 3);
        half[turn_at(part, 1)] = __builtin_shufflevector(x.p[part], x.p[part], 4, 5, 6, 7);
      }
      add_columns<DH>(dv, gt, 0, lane, split_pair(s));
      add_columns<DH>(dk, qt, 0, lane, x);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) {
      const int n = (wave * (DH / 32) + i) / 2, h = (wave * (DH / 32) + i) % 2;
      f32x4 dq[1] = {zero4()};
#pragma unroll 1
      for (int first = 0; first < len; first += 32)
        dq[0] = product6(Tile<DH>::columns(kt, first, n, lane), Turn::columns(turn, first, h, lane), dq[0]);
      const int row = t + 16 * h + c;
      if (row < r1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) dq[0][e] *= kLn2;
        store_quad(p.dq.ptr + row_offset(p, p.dq.ld, b, hk, row), 16 * n + 4 * g, p.dh, p.vec, dq[0]);
      }
    }
  }
  if (key >= p.Nk) return;
  if (!key_ok) {  // (whatever its column held)
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) dk[n] = zero4(), dv[n] = zero4();
  }
  if (p.splits > 1) {
    const long long pitch = (long long)p.Hkv * p.dh, all = (long long)p.B * p.Nk * pitch;
    const long long at = key_offset(p, pitch, b, hk, key);
    store_row<DH>(p.part + split * all + at, dk, p.scale, g, p.dh, p.dh % 4 == 0);
    store_row<DH>(p.part + (p.splits + split) * all + at, dv, 1.f, g, p.dh, p.dh % 4 == 0);
  } else {
    store_row<DH>(p.dk.ptr + key_offset(p, p.dk.ld, b, hk, key), dk, p.scale, g, p.dh, p.vec);
    store_row<DH>(p.dv.ptr + key_offset(p, p.dv.ld, b, hk, key), dv, 1.f, g, p.dh, p.vec);
  }
}

// out[row][col] = sum of the parts in order; `rows` rows of `width` columns; of two gradients at once: y
__global__ __launch_bounds__(256) void cross_add_parts_kernel(const float *part, int splits, long long rows, int width,
                                                              Result x, Result y) {
  const long long all = rows * width;
  const Result out = blockIdx.y == 0 ? x : y;
  part += blockIdx.y * splits * all;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 4
    for (int x = 0; x < splits; ++x) s += part[x * all + i];
    const long long r = i / width;
    out.ptr[r * out.ld + (i - r * width)] = s;
  }
}

// Groups of 16 in a workgroup, blocks, and how the other side is split.
struct Side {
  Block block;
  int blocks, splits, chunk;
};
Side plan_side(long long own, long long other, long long heads, int dh, bool keys, double part_us) {
  Side s;
  s.block = plan_block(own, other, heads, dh <= 96, keys ? 0 : 1024, keys ? 64 : 128);
  // Up to 32 keys, or rows of wide heads: eight waves, half of which only load (668 x 14 x 128, 24 key heads: 109 -> 88 us,
  // 98 x 24 x 80, 128: 49 -> 41; rows: 10 x 814 x 128, 42 heads: 94 -> 74; of 80 columns no difference).
  if (own <= 32 && (keys || dh > 96)) s.block = {4, 8};
  const int groups = s.block.groups;
  s.blocks = (int)((own + 16 * groups - 1) / (16 * groups));
  const long long stages = (other + 63) / 64;
  const int wide = dh <= 32 ? 32 : dh <= 64 ? 64 : dh <= 96 ? 96 : 128;
  const int four = keys ? 2 : dq_resident(dh);
  const int resident = groups == 4 && s.block.waves == 4 ? four : groups == 2 ? 2 : 1;  // workgroups a CU
  const double flop = 32.0 * (keys ? 4 : 3) * groups * other * wide;  // of a block; 0.5 TFLOP/s a CU
  const int splits = plan_splits(heads * s.blocks, resident * (long long)vitk::cu_count(), stages,
                                 flop / (0.5e6 / resident), 3.0 * wide / 64, part_us);
  s.chunk = std::max((int)((stages + splits - 1) / splits) * 64, 64);
  s.splits = std::max((int)((other + s.chunk - 1) / s.chunk), 1);
  return s;
}
struct Plan {
  Side rows, keys;
  bool few_keys;       // one kernel for all gradients
  size_t delta, part;  // floats
};
Plan make_plan(const Params &p) {
  Plan n;
  const long long heads = (long long)p.B * p.Hkv;
  // one part of the results, written and read at 4 TB/s
  n.rows = plan_side(p.rows, p.Nk, heads, p.dh, false, 2.0 * p.B * p.H * p.Nq * p.dh * 4 / 4e6);
  n.keys = plan_side(p.Nk, p.rows, heads, p.dh, true, 4.0 * p.B * p.Hkv * p.Nk * p.dh * 4 / 4e6);
  n.few_keys = p.Nk > 0 && p.Nk <= FEW_KEYS && p.dh <= 64;
  if (n.few_keys) {  // one round of workgroups, and two stages of rows or more in each
    const long long stages = ((long long)p.rows + 31) / 32;
    const long long places = short_resident(p.dh) * (long long)vitk::cu_count();
    const int splits = (int)std::max(std::min({places / heads, (stages + 1) / 2, (long long)16}), 1ll);
    n.keys.blocks = 1;
    n.keys.chunk = std::max((int)((stages + splits - 1) / splits) * 32, 32);
    n.keys.splits = std::max((int)(((long long)p.rows + n.keys.chunk - 1) / n.keys.chunk), 1);
  }
  n.delta = n.few_keys ? 0 : ((size_t)p.B * p.H * p.Nq + 63) / 64 * 64;
  const size_t q = !n.few_keys && n.rows.splits > 1 ? (size_t)n.rows.splits * p.B * p.Nq * p.H * p.dh : 0;
  const size_t k = n.keys.splits > 1 ? (size_t)2 * n.keys.splits * p.B * p.Nk * p.Hkv * p.dh : 0;
  n.part = std::max(q, k);  // one after the other
  return n;
}

template <int DH>
void launch_dq(const Params &p, Block block, unsigned wgs, hipStream_t st) {
  if constexpr (DH <= 96) {
    if (block.groups == 4 && block.waves == 4) {
      hipLaunchKernelGGL((cross_dq_kernel<DH, 4, 4>), dim3(wgs), dim3(256), 0, st, p);
      return;
    }
  }
  if (block.groups == 8)
    hipLaunchKernelGGL((cross_dq_kernel<DH, 8, 8>), dim3(wgs), dim3(512), 0, st, p);
  else if (DH > 96 || block.groups == 4)
    hipLaunchKernelGGL((cross_dq_kernel<DH, 8, 4>), dim3(wgs), dim3(512), 0, st, p);
  else if constexpr (DH <= 96)
    hipLaunchKernelGGL((cross_dq_kernel<DH, 4, 2>), dim3(wgs), dim3(256), 0, st, p);
}
template <int DH>
void launch_dkv(const Params &p, Block block, unsigned wgs, hipStream_t st) {
  if constexpr (DH > 64) {  // others are not here with so few keys
    if (block.groups == 4 && block.waves == 8) {
      hipLaunchKernelGGL((cross_dkv_kernel<DH, 8, 4>), dim3(wgs), dim3(512), 0, st, p);
      return;
    }
  }
  if constexpr (DH <= 96) {
    if (block.groups == 4) {
      hipLaunchKernelGGL((cross_dkv_kernel<DH, 4, 4>), dim3(wgs), dim3(256), 0, st, p);
      return;
    }
  }
  hipLaunchKernelGGL((cross_dkv_kernel<DH, 8, 8>), dim3(wgs), dim3(512), 0, st, p);
}
void add_parts(const float *part, int splits, long long rows, int width, Result x, const Result *y, hipStream_t st) {
  hipLaunchKernelGGL(cross_add_parts_kernel, dim3(vitk::grid_for(rows * width, 256), y ? 2 : 1), dim3(256), 0, st, part,
                     splits, rows, width, x, y ? *y : x);
}

template <int DH>
int launch(Params p, const Plan &n, hipStream_t st) {
  const long long heads = (long long)p.B * p.Hkv;
  const long long qw = heads * n.rows.blocks * n.rows.splits, kw = heads * n.keys.blocks * n.keys.splits;
  VITK_REQUIRE((n.few_keys || vitk::fits_one_launch(qw, DH > 96 ? 512 : 64 * n.rows.block.waves)) &&
                   vitk::fits_one_launch(kw, n.few_keys ? 256 : 64 * n.keys.block.waves),
               "vitk_cross_sdpa_bwd: too many rows for one launch");
  if (p.Nq > 0 && !n.few_keys) {
    p.blocks = n.rows.blocks, p.splits = n.rows.splits, p.chunk = n.rows.chunk;
    launch_dq<DH>(p, n.rows.block, (unsigned)qw, st);
    if (p.splits > 1) add_parts(p.part, p.splits, (long long)p.B * p.Nq, p.H * p.dh, p.dq, nullptr, st);
  }
  if (p.Nk > 0) {
    p.blocks = n.keys.blocks, p.splits = n.keys.splits, p.chunk = n.keys.chunk;
    if (n.few_keys) {
      if constexpr (DH <= 64) hipLaunchKernelGGL(cross_short_kernel<DH>, dim3((unsigned)kw), dim3(256), 0, st, p);
    } else {
      launch_dkv<DH>(p, n.keys.block, (unsigned)kw, st);
    }
    if (p.splits > 1) add_parts(p.part, p.splits, (long long)p.B * p.Nk, p.Hkv * p.dh, p.dk, &p.dv, st);
  }
  return vitk::check_launch("vitk_cross_sdpa_bwd");
}

}  // namespace

extern "C" size_t vitk_cross_sdpa_bwd_workspace_bytes(const vitk_cross_sdpa_args *a) {
  if (!a || a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->Nq < 0 || a->Nk < 0 || a->dh < 1 ||
      !few_enough_rows(a))
    return 0;
  Params p = {};
  p.B = a->B, p.H = a->H, p.Hkv = a->Hkv, p.G = a->H / a->Hkv, p.Nq = a->Nq, p.Nk = a->Nk, p.dh = a->dh;
  p.rows = p.G * p.Nq;
  const Plan n = make_plan(p);
  return (n.delta + n.part) * sizeof(float);
}

extern "C" int vitk_cross_sdpa_bwd(const vitk_cross_sdpa_args *a, vitk_stream_t stream) {
  Params p = {};
  if (check_args("vitk_cross_sdpa_bwd", a, true, &p)) return 1;
  if (p.B == 0 || (p.Nq == 0 && p.Nk == 0)) return 0;
  const Plan n = make_plan(p);
  const size_t need = (n.delta + n.part) * sizeof(float);
  VITK_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need),
               "vitk_cross_sdpa_bwd: workspace of %zu bytes needed, %zu given", need, a->workspace ? a->workspace_bytes : 0);
  VITK_REQUIRE(need == 0 || vitk::aligned16(a->workspace), "vitk_cross_sdpa_bwd: workspace is not 16-byte aligned");
  p.delta = a->workspace;
  p.part = a->workspace + n.delta;
  hipStream_t st = vitk::as_stream(stream);
  if (p.dh <= 32) return launch<32>(p, n, st);
  if (p.dh <= 64) return launch<64>(p, n, st);
  if (p.dh <= 96) return launch<96>(p, n, st);
  return launch<128>(p, n, st);
}
