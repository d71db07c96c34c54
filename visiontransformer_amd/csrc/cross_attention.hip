// Cross attention forward: softmax(scale * q k^T) v with queries and keys of different sequences.
//
// One workgroup = up to 128 query rows of one (batch, key head); the query heads that share the key head are
// rows of the same block, so shared keys are read once per block.  A wave holds 16 rows as the columns of
// S^T[key][row] = K Q^T; what a lane receives of 32 keys is the operand that the second product
// O^T[d][row] += V^T P^T wants from it, so probabilities never leave their registers.  One pass over the
// keys with a running maximum and sum per row.
//
// Bounds: the matrix cores where keys are many (1021 x 4099 x 64, 48 heads: 200 - 220 us for 38.6 GFLOP, six bf16
// products each, 1050 - 1160 TFLOP/s of them; 512 x 1536 x 96, 128 heads: 239 us, 970), the loads and splits of
// a stage where they are few (48 x 197 x 64, 768 heads: 24.7 us, 3.9 TB/s), memory for a few rows.
#include "cross_attention.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace vitk {
namespace cross {

int check_args(const char *who, const vitk_cross_sdpa_args *a, bool backward, Params *p) {
  VITK_REQUIRE(a != nullptr, "%s: null arguments", who);
  VITK_REQUIRE(a->reserved == 0, "%s: reserved must be 0", who);
  VITK_REQUIRE(a->B >= 0 && a->Nq >= 0 && a->Nk >= 0, "%s: negative size", who);
  VITK_REQUIRE(a->H > 0 && a->Hkv > 0 && a->H % a->Hkv == 0, "%s: %d query heads over %d key heads", who, a->H, a->Hkv);
  VITK_REQUIRE(a->dh >= 1 && a->dh <= 128, "%s: head dimension %d outside [1, 128]", who, a->dh);
  VITK_REQUIRE(std::isfinite(a->scale), "%s: scale is not a finite number", who);
  const long long wq = (long long)a->H * a->dh, wk = (long long)a->Hkv * a->dh;
  const bool any_q = a->B > 0 && a->Nq > 0, any_k = a->B > 0 && a->Nk > 0;
  VITK_REQUIRE(few_enough_rows(a), "%s: too many rows", who);
  if (any_q) {
    VITK_REQUIRE(a->q && a->out, "%s: null pointer", who);
    VITK_REQUIRE(a->ld_q >= wq && a->ld_out >= wq, "%s: row pitch below H*dh", who);
  }
  if (any_k) {
    VITK_REQUIRE(a->k && a->v, "%s: null pointer", who);
    VITK_REQUIRE(a->ld_k >= wk && a->ld_v >= wk, "%s: row pitch below Hkv*dh", who);
  }
  const float *in[] = {a->q, a->k, a->v};
  auto fresh = [&](const float *out) {  // not one of the inputs
    bool ok = true;
    for (const float *x : in) ok = ok && (out == nullptr || out != x);
    return ok;
  };
  VITK_REQUIRE(fresh(a->out), "%s: out is one of the inputs", who);
  p->q = {a->q, a->ld_q};
  p->k = {a->k, a->ld_k};
  p->v = {a->v, a->ld_v};
  p->out = {a->out, a->ld_out};
  p->o = {a->out, a->ld_out};
  p->len = a->key_len;
  p->stats = a->stats;
  p->B = a->B, p->H = a->H, p->Hkv = a->Hkv, p->G = a->H / a->Hkv, p->Nq = a->Nq, p->Nk = a->Nk, p->dh = a->dh;
  p->rows = p->G * p->Nq;
  p->scale = a->scale, p->c = a->scale * kLog2e;
  bool vec = a->dh % 4 == 0;
  auto quad = [&](const void *ptr, int64_t ld) { vec = vec && aligned16(ptr) && ld % 4 == 0; };
  quad(a->q, a->ld_q), quad(a->k, a->ld_k), quad(a->v, a->ld_v), quad(a->out, a->ld_out);
  if (backward) {
    if (any_q) {
      VITK_REQUIRE(a->dout && a->dq && a->stats, "%s: null pointer", who);
      VITK_REQUIRE(a->ld_dout >= wq && a->ld_dq >= wq, "%s: row pitch below H*dh", who);
    }
    if (any_k) {
      VITK_REQUIRE(a->dk && a->dv, "%s: null pointer", who);
      VITK_REQUIRE(a->ld_dk >= wk && a->ld_dv >= wk, "%s: row pitch below Hkv*dh", who);
    }
    for (const float *x : {a->dq, a->dk, a->dv})
      VITK_REQUIRE(fresh(x) && (x == nullptr || (x != a->out && x != a->dout)), "%s: a gradient is one of the inputs", who);
    VITK_REQUIRE(!a->dk || (a->dk != a->dv && a->dk != a->dq), "%s: two gradients share a buffer", who);
    VITK_REQUIRE(!a->dq || a->dq != a->dv, "%s: two gradients share a buffer", who);
    p->dout = {a->dout, a->ld_dout};
    p->dq = {a->dq, a->ld_dq};
    p->dk = {a->dk, a->ld_dk};
    p->dv = {a->dv, a->ld_dv};
    quad(a->dout, a->ld_dout), quad(a->dq, a->ld_dq), quad(a->dk, a->ld_dk), quad(a->dv, a->ld_dv);
  }
  p->vec = vec;
  return 0;
}

}  // namespace cross
}  // namespace vitk

namespace {

using namespace vitk::cross;

// NW waves: RW groups of 16 rows, and NW / RW waves that share such a group's keys (few rows: the keys of a
// stage are dealt to the waves instead of leaving them idle; their results are joined in LDS).
// Blocks of 64 rows as four waves of 16, whose keys no waves share: with one buffer up to four such workgroups are
// on a CU and hide each other's loads and barriers.  48 rows x 197 keys x 64, 768 heads: 24.7 us; eight waves
// that share the keys took 4 us more.
constexpr int waves_a_simd(int dh, int nw, int rw) {
  if (nw == rw) return dh <= 64 ? 4 : nw == 8 ? (dh <= 96 ? 4 : 2) : dh <= 96 ? 3 : 2;
  return nw == 8 ? (dh <= 64 ? 4 : 2) : dh <= 64 ? 2 : 1;
}
template <int DH, int NW, int RW>
__global__ __launch_bounds__(64 * NW, waves_a_simd(DH, NW, RW)) void cross_fwd_kernel(const Params p) {
  typedef Shape<DH, NW, RW> S;
  constexpr int NB = DH / 16, BOX = DH / 4 + 2;  // words a lane passes on: o, m, l
  constexpr int JOIN = S::OTHER > 1 ? RW * 64 * BOX * 4 : 0;
  __shared__ __attribute__((aligned(16))) char lds[2 * S::BUFFERS * S::UNITS * 16 > JOIN ? 2 * S::BUFFERS * S::UNITS * 16 : JOIN];
  bf16x8 *buffers = reinterpret_cast<bf16x8 *>(lds);
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rg = wave % RW, kg = wave / RW;
  long long wg = blockIdx.x;
  const int rb = (int)(wg % p.blocks);
  wg /= p.blocks;
  const int hk = (int)(wg % p.Hkv);
  wg /= p.Hkv;
  const int b = (int)(wg % p.B), split = (int)(wg / p.B);
  const int len = valid_keys(p, b);
  const int k0 = min((long long)split * p.chunk, (long long)len), k1 = min((long long)k0 + p.chunk, (long long)len);
  const int row = (rb * RW + rg) * 16 + c;
  const bool row_ok = row < p.rows;

  Split8 q[DH / 32];  // times scale log2(e)
  float raw[DH / 32][8];
  load_raw<DH>(raw, p.q.ptr + row_offset(p, p.q.ld, b, hk, row_ok ? row : 0), g, p);
  f32x4 o[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) o[n] = zero4();
  float m = 0.f, l = 0.f;
  bool started = false;  // (uniform)

  Stage<DH, NW, RW> next;
  auto at = [&](bool y, int n) {
    return y ? p.v.ptr + key_offset(p, p.v.ld, b, hk, n) : p.k.ptr + key_offset(p, p.k.ld, b, hk, n);
  };
  const bool early = wave < NW / 2, empty = (rb * RW + rg) * 16 >= p.rows;
  next.fetch(p, k0, k1, at);
  split_row<DH>(q, raw, row_ok, p.c);
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
    const int first = 32 * kg;  // of the stage
    if (!empty && t + first < k1) {
      f32x4 s[2] = {all4(-m), all4(-m)};  // the products are added to this: what the exponent wants
      rows_times<DH>(kt, first, c, g, q, s);
      if (t + first + 32 > k1) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t + first + 16 * h + 4 * g + e >= k1) s[h][e] = -INFINITY;
      }
      float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int e = 1; e < 4; ++e) top = fmaxf(top, fmaxf(s[0][e], s[1][e]));
      top = column_max(top);
      if (!started || __any(top > 0.f)) {
        const float up = started ? fmaxf(top, 0.f) : top, fall = started ? __builtin_amdgcn_exp2f(-up) : 0.f;
        m += up;
        l *= fall;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= fall;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[h][e] -= up;
        started = true;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][e] = __builtin_amdgcn_exp2f(s[h][e]);
          l += s[h][e];  // of this lane's quarter of the keys
        }
      add_columns<DH>(o, vt, first, lane, split_pair(s));
    }
    if (S::BUFFERS == 2 && !early) advance();
    __syncthreads();
  }
  l = column_sum(l);
  if (!started) m = -INFINITY;
  if constexpr (S::OTHER > 1) {
    static_assert(S::OTHER == 2, "two key groups");
    float *box = reinterpret_cast<float *>(lds) + rg * 64 * BOX + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) box[(4 * n + e) * 64] = o[n][e];
      box[(BOX - 2) * 64] = m;
      box[(BOX - 1) * 64] = l;
    }
    __syncthreads();
    if (kg == 1) return;
    const float m2 = box[(BOX - 2) * 64], l2 = box[(BOX - 1) * 64], top = fmaxf(m, m2);
    if (top > -INFINITY) {
      const float f1 = __builtin_amdgcn_exp2f(m - top), f2 = __builtin_amdgcn_exp2f(m2 - top);
      l = l * f1 + l2 * f2;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = o[n][e] * f1 + box[(4 * n + e) * 64] * f2;
      m = top;
    }
  }
  if (!row_ok) return;
  const long long stat = row_stat(p, b, hk, row);
  float *dst, *st;
  float f = 1.f;
  bool vec = p.vec;
  if (p.splits > 1) {
    const long long all = (long long)p.B * p.H * p.Nq;
    dst = p.part + (split * all + stat) * p.dh;
    st = p.part + p.splits * all * p.dh + (split * all + stat) * 2;
    vec = p.dh % 4 == 0;
  } else {
    dst = p.out.ptr + row_offset(p, p.out.ld, b, hk, row);
    st = p.stats ? p.stats + stat * 2 : nullptr;
    f = l == 0.f ? 0.f : 1.f / l;
    if (l == 0.f) m = 0.f;
  }
  store_row<DH>(dst, o, f, g, p.dh, vec);
  if (st && g == 0) {
    st[0] = m;
    st[1] = l;
  }
}

constexpr int JOIN_FEW = 8, JOIN_WAVES = 16, MAX_SPLITS = 64 * JOIN_WAVES;
// Joins up to eight parts of split rows: LP lanes per row, four columns each, all parts in flight.
template <int LP>
__global__ __launch_bounds__(256) void cross_join_kernel(const Params p) {
  const long long all = (long long)p.B * p.H * p.Nq;
  const long long r = (blockIdx.x * 256ll + threadIdx.x) / LP;
  if (r >= all) return;
  const int d = threadIdx.x % LP * 4;
  const bool vec = p.dh % 4 == 0;
  const float *st = p.part + p.splits * all * p.dh + 2 * r, *src = p.part + r * p.dh;
  float ms[JOIN_FEW], ls[JOIN_FEW], m = -INFINITY, l = 0.f;
  f32x4 x[JOIN_FEW], o = zero4();
#pragma unroll
  for (int s = 0; s < JOIN_FEW; ++s) {
    ms[s] = -INFINITY, ls[s] = 0.f, x[s] = zero4();
    if (s < p.splits) {
      ms[s] = st[s * all * 2], ls[s] = st[s * all * 2 + 1];
      x[s] = load_quad(src + s * all * p.dh, d, p.dh, vec);
    }
  }
#pragma unroll
  for (int s = 0; s < JOIN_FEW; ++s) m = fmaxf(m, ms[s]);
  if (m == -INFINITY) m = 0.f;  // no key at all
#pragma unroll
  for (int s = 0; s < JOIN_FEW; ++s) {
    const float f = __builtin_amdgcn_exp2f(ms[s] - m);
    l += f * ls[s];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += f * x[s][e];
  }
  const float scale = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= scale;
  const long long bh = r / p.Nq, n = r % p.Nq, b = bh / p.H, h = bh % p.H;
  store_quad(p.out.ptr + (b * p.Nq + n) * p.out.ld + h * p.dh, d, p.dh, p.vec, o);
  if (d == 0 && p.stats) {
    p.stats[2 * r] = m;
    p.stats[2 * r + 1] = l;
  }
}

// More than eight parts (few rows): W waves per row, each joins up to 64 parts, a lane per part for the statistics,
// then lanes over the columns; every part's statistics arrive in one round trip (49 parts of 256 rows: 4.8 us, in
// batches of eight 23).
template <int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void cross_join_many_kernel(const Params p) {
  __shared__ float box[W][130];
  const long long all = (long long)p.B * p.H * p.Nq;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long r = W == 1 ? blockIdx.x * 4ll + wave : blockIdx.x;
  if (r >= all) return;
  const int per = (p.splits + W - 1) / W, s0 = W == 1 ? 0 : min(wave * per, p.splits), s1 = min(s0 + per, p.splits);
  const float *st = p.part + p.splits * all * p.dh;
  float m = -INFINITY, l = 0.f;
  if (s0 + lane < s1) {
    m = st[((s0 + lane) * all + r) * 2];
    l = st[((s0 + lane) * all + r) * 2 + 1];
  }
  float top = vitk::wave_max(m);
  if constexpr (W > 1) {
    if (lane == 0) box[wave][0] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, box[w][0]);
    __syncthreads();
  }
  if (top == -INFINITY) top = 0.f;  // no key at all
  const float f = __builtin_amdgcn_exp2f(m - top);
  l = vitk::wave_sum(l * f);
  float x0 = 0.f, x1 = 0.f;
  const float *src = p.part + r * p.dh + lane;
  for (int s = s0; s < s1; s += 8) {  // eight parts in flight
    float a[8], b[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool in = s + u < s1;
      a[u] = in && lane < p.dh ? src[(s + u) * all * p.dh] : 0.f;
      b[u] = in && lane + 64 < p.dh ? src[(s + u) * all * p.dh + 64] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float fs = __shfl(f, (s - s0 + u) & 63, 64);  // (parts behind the last one: 0 times something finite)
      x0 += fs * a[u];
      x1 += fs * b[u];
    }
  }
  if constexpr (W > 1) {
    box[wave][lane] = x0, box[wave][64 + lane] = x1;
    if (lane == 0) box[wave][128] = l;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) x0 += box[w][lane], x1 += box[w][64 + lane], l += box[w][128];
  }
  const float scale = l == 0.f ? 0.f : 1.f / l;
  const long long bh = r / p.Nq, n = r % p.Nq, b = bh / p.H, h = bh % p.H;
  float *dst = p.out.ptr + (b * p.Nq + n) * p.out.ld + h * p.dh;
  if (lane < p.dh) dst[lane] = x0 * scale;
  if (lane + 64 < p.dh) dst[lane + 64] = x1 * scale;
  if (lane == 0 && p.stats) {
    p.stats[2 * r] = top;
    p.stats[2 * r + 1] = l;
  }
}

// ------------------------------------------------------------------------------------- few rows
// At most 4 rows per key head, 8 of wide heads (single tokens): every key and value is read once and used for a few
// dot products, so memory bounds this and the vector ALU computes it.  LP lanes share a key, four columns each;
// 64 / LP keys per wave and U of those in flight: fewer for more rows, since more waves a SIMD read faster than more
// loads in fewer waves.  16 x 12345 keys x 4 heads x 128, 809 MB: one row 121 us = 6.7 TB/s, four rows 131.
// Each batch entry is cut into equal parts, so ragged lengths leave no workgroup without work.  Each group of
// LP lanes keeps a running maximum and sum per row of its own; groups, then waves, are joined at the end.
template <int LP>
__device__ __forceinline__ float group_sum(float x) {  // over LP neighbouring lanes, in all of them
  auto add = [&](auto ctrl) {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl.value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0xB1>());   // neighbours
  add(std::integral_constant<int, 0x4E>());   // pairs
  add(std::integral_constant<int, 0x141>());  // mirrored halves of a row of 16
  if constexpr (LP >= 16) add(std::integral_constant<int, 0x140>());  // mirrored rows
  if constexpr (LP >= 32)  // lane ^ 16
    x += __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), 0x401F));
  return x;
}

template <int LP, int R, int NW>
__global__ __launch_bounds__(64 * NW) void cross_row_kernel(const Params p) {
  constexpr int U = R <= 2 ? 4 : 2, KEYS = 64 / LP, DP = 4 * LP;
  __shared__ float box[NW][R][DP + 2];
  const int lane = threadIdx.x & 63, li = lane % LP, lg = lane / LP, d = 4 * li;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  long long wg = blockIdx.x;
  const int hk = (int)(wg % p.Hkv);
  wg /= p.Hkv;
  const int b = (int)(wg % p.B), split = (int)(wg / p.B);
  const int len = valid_keys(p, b);
  const int chunk = (len / p.splits + 16) / 16 * 16;  // each batch entry in equal parts
  const int k0 = min((long long)split * chunk, (long long)len), k1 = min((long long)k0 + chunk, (long long)len);
  f32x4 q[R], o[R];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    q[r] = o[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[r] = -INFINITY, l[r] = 0.f;
    if (r < p.rows) {
      q[r] = load_quad(p.q.ptr + row_offset(p, p.q.ld, b, hk, r), d, p.dh, p.vec);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[r][e] *= p.c;
    }
  }
  const float *kp = p.k.ptr + key_offset(p, p.k.ld, b, hk, 0), *vp = p.v.ptr + key_offset(p, p.v.ld, b, hk, 0);
  const int first = d < p.dh ? d : 0;
  for (int t = k0 + wave * KEYS * U; t < k1; t += NW * KEYS * U) {
    // Keys behind the end stand for the last one, with a score of -inf; columns behind dh meet zeros of q, and
    // nobody reads their sums.  (Nontemporal: nobody reads a key again.)
    f32x4 k[U], v[U];
    if (p.vec) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = min(t + u * KEYS + lg, k1 - 1);
        k[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(kp + key * p.k.ld + first));
        v[u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(vp + key * p.v.ld + first));
      }
    } else {
      int from = d;
      asm volatile("" : "+v"(from));  // (the compiler would keep these places in registers for the whole loop)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = min(t + u * KEYS + lg, k1 - 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          k[u][e] = kp[key * p.k.ld + min(from + e, p.dh - 1)];
          v[u][e] = vp[key * p.v.ld + min(from + e, p.dh - 1)];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[U], top = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = group_sum<LP>((q[r][0] * k[u][0] + q[r][1] * k[u][1]) + (q[r][2] * k[u][2] + q[r][3] * k[u][3]));
        if (t + u * KEYS + lg >= k1) s[u] = -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float base = top == -INFINITY ? 0.f : top, fall = __builtin_amdgcn_exp2f(m[r] - base);
      m[r] = top;
      l[r] *= fall;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] *= fall;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float x = __builtin_amdgcn_exp2f(s[u] - base);
        l[r] += x;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[r][e] += x * v[u][e];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int off = LP; off < 64; off <<= 1) {
      const float m2 = __shfl_xor(m[r], off, 64), l2 = __shfl_xor(l[r], off, 64);
      const float top = fmaxf(m[r], m2), base = top == -INFINITY ? 0.f : top;
      const float f1 = __builtin_amdgcn_exp2f(m[r] - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
      l[r] = l[r] * f1 + l2 * f2;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][e] = o[r][e] * f1 + __shfl_xor(o[r][e], off, 64) * f2;
      m[r] = top;
    }
    if (lg == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) box[wave][r][d + e] = o[r][e];
      if (li == 0) box[wave][r][DP] = m[r], box[wave][r][DP + 1] = l[r];
    }
  }
  __syncthreads();
  const long long all = (long long)p.B * p.H * p.Nq;
  for (int i = threadIdx.x; i < R * DP; i += 64 * NW) {
    const int r = i / DP, col = i % DP;
    if (r >= p.rows || col >= p.dh) continue;
    float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, box[w][r][DP]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(box[w][r][DP] - base);
      sum += f * box[w][r][DP + 1];
      x += f * box[w][r][col];
    }
    const long long stat = row_stat(p, b, hk, r);
    if (p.splits > 1) {
      p.part[(split * all + stat) * p.dh + col] = x;
      float *st = p.part + p.splits * all * p.dh + (split * all + stat) * 2;
      if (col == 0) st[0] = top, st[1] = sum;
    } else {
      p.out.ptr[row_offset(p, p.out.ld, b, hk, r) + col] = sum == 0.f ? 0.f : x / sum;
      if (col == 0 && p.stats) p.stats[2 * stat] = base, p.stats[2 * stat + 1] = sum;
    }
  }
}

// The kernel, the rows of a workgroup, and over how many workgroups the keys of a block are split.
constexpr int CHUNK = 64;      // key ranges of splits are multiples of this
// Rows per key head up to which the vector kernel runs (eight rows, 320 heads x 1000 keys: of 64 columns 53 us, the
// matrix kernel 38; of 128 columns 100 and 133).
constexpr int few_rows(int dh) { return dh <= 96 ? 4 : 8; }
struct FwdPlan {
  Block block;  // no groups = the vector kernel
};
FwdPlan plan_fwd(Params *p) {
  FwdPlan f = {};
  const long long heads = (long long)p->B * p->Hkv, stages = ((long long)p->Nk + CHUNK - 1) / CHUNK;
  long long splits = 1;
  if (p->rows <= few_rows(p->dh)) {
    p->blocks = 1;
    f.block.waves = 4;
    // One round of the workgroups that fit the device by their registers, 64 keys or more each (16 x 12345 keys x 4
    // heads x 128, four rows, ragged: 117 us with 5 a CU, 126 in 39 parts whatever fits; 48 x 12 heads x 3000 x 64, one
    // row: 142 us in three parts, 223 in one; 2 x 100000 keys x 2 heads 67, in at most 64 parts 209; one batch entry
    // of 4000 keys x 8 heads x 64: 15 us in parts of 64 keys, 20 in parts of 256).
    const long long cus = vitk::cu_count(), places = cus * (p->rows <= 2 ? 7 : p->rows <= 4 ? 5 : 4);
    const int few = p->rows == 1 ? 448 : p->rows <= 4 ? 320 : 192;  // keys
    if (p->Nk <= few && heads <= (p->rows == 1 ? 2 * cus : cus))
      f.block.waves = 16;  // one launch (515 keys, 40 heads of 80, one row: 18 us, in parts 15; 260 keys: 7 and 9)
    else if (heads > 0)
      splits = std::min(places / heads, stages);
  } else {
    // A workgroup of 64 rows with one buffer is worth its empty waves even for 9 to 32 rows: more of them are on a
    // CU (16 x 1000, 320 heads of 64: 49 -> 38 us, of 128: 220 -> 133; of 32 no difference).
    f.block = plan_block(p->rows, p->Nk, heads, true, p->dh <= 96 ? 1024 : 512, 0);
    const long long cus = vitk::cu_count();
    if (p->rows <= 32 && p->dh > 32 && 4 * heads >= cus && heads * stages >= cus) f.block = {4, 4};
    const int groups = f.block.groups;
    p->blocks = (int)(((long long)p->rows + 16 * groups - 1) / (16 * groups));
    const int wide = p->dh <= 32 ? 32 : p->dh <= 64 ? 64 : p->dh <= 96 ? 96 : 128;
    const int resident = groups == 4 && f.block.waves == 4 ? waves_a_simd(wide, 4, 4)  // workgroups a CU
                                                           : (groups == 2 ? 2 : 1) * (wide <= 96 ? 2 : 1);
    const double flop = 64.0 * groups * p->Nk * wide;                 // of a block; 0.6 TFLOP/s a CU
    const double part = 2.0 * p->B * p->H * p->Nq * p->dh * 4 / 4e6;  // written and read at 4 TB/s
    splits = vitk::cross::plan_splits(heads * p->blocks, resident * (long long)vitk::cu_count(), stages,
                                      flop / (0.6e6 / resident), 3.0 * wide / 64, part);
  }
  if (splits > MAX_SPLITS) splits = MAX_SPLITS;
  if (splits < 1) splits = 1;
  if (f.block.groups == 0) {
    p->splits = (int)splits;  // each batch entry in that many equal parts
    return f;
  }
  p->chunk = (int)((stages + splits - 1) / splits) * CHUNK;
  if (p->chunk == 0) p->chunk = CHUNK;
  p->splits = (int)(((long long)p->Nk + p->chunk - 1) / p->chunk);
  if (p->splits < 1) p->splits = 1;
  return f;
}

template <int LP, int NW>
void launch_rows(const Params &p, unsigned wgs, hipStream_t st) {
  const dim3 grid(wgs), block(64 * NW);
  if (p.rows == 1)
    hipLaunchKernelGGL((cross_row_kernel<LP, 1, NW>), grid, block, 0, st, p);
  else if (p.rows == 2)
    hipLaunchKernelGGL((cross_row_kernel<LP, 2, NW>), grid, block, 0, st, p);
  else if (p.rows <= 4)
    hipLaunchKernelGGL((cross_row_kernel<LP, 4, NW>), grid, block, 0, st, p);
  else if constexpr (LP == 32)  // (narrower heads are not here with more)
    hipLaunchKernelGGL((cross_row_kernel<LP, 8, NW>), grid, block, 0, st, p);
}
template <int LP>
void launch_rows(const Params &p, int waves, unsigned wgs, hipStream_t st) {
  if (waves == 4)
    launch_rows<LP, 4>(p, wgs, st);
  else
    launch_rows<LP, 16>(p, wgs, st);
}

template <int DH>
void launch_fwd(const Params &p, Block block, unsigned wgs, hipStream_t st) {
  if (block.groups == 8)
    hipLaunchKernelGGL((cross_fwd_kernel<DH, 8, 8>), dim3(wgs), dim3(512), 0, st, p);
  else if (block.groups == 4 && block.waves == 8)
    hipLaunchKernelGGL((cross_fwd_kernel<DH, 8, 4>), dim3(wgs), dim3(512), 0, st, p);
  else if (block.groups == 4)
    hipLaunchKernelGGL((cross_fwd_kernel<DH, 4, 4>), dim3(wgs), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((cross_fwd_kernel<DH, 4, 2>), dim3(wgs), dim3(256), 0, st, p);
}

size_t fwd_bytes(const Params &p) {
  if (p.splits <= 1) return 0;
  return (size_t)p.splits * p.B * p.H * p.Nq * (p.dh + 2) * sizeof(float);
}

}  // namespace

extern "C" size_t vitk_cross_sdpa_fwd_workspace_bytes(const vitk_cross_sdpa_args *a) {
  if (!a || a->B <= 0 || a->Nq <= 0 || a->Nk < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->dh < 1 || !few_enough_rows(a))
    return 0;
  Params p = {};
  p.B = a->B, p.H = a->H, p.Hkv = a->Hkv, p.G = a->H / a->Hkv, p.Nq = a->Nq, p.Nk = a->Nk, p.dh = a->dh;
  p.rows = p.G * p.Nq;
  plan_fwd(&p);
  return fwd_bytes(p);
}

extern "C" int vitk_cross_sdpa_fwd(const vitk_cross_sdpa_args *a, vitk_stream_t stream) {
  Params p = {};
  if (check_args("vitk_cross_sdpa_fwd", a, false, &p)) return 1;
  if (p.B == 0 || p.Nq == 0) return 0;
  const FwdPlan plan = plan_fwd(&p);
  const size_t need = fwd_bytes(p);
  VITK_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need),
               "vitk_cross_sdpa_fwd: workspace of %zu bytes needed, %zu given", need, a->workspace ? a->workspace_bytes : 0);
  VITK_REQUIRE(need == 0 || vitk::aligned16(a->workspace), "vitk_cross_sdpa_fwd: workspace is not 16-byte aligned");
  p.part = a->workspace;
  const long long wgs = (long long)p.B * p.Hkv * p.blocks * p.splits;
  const long long rows = (long long)p.B * p.H * p.Nq;  // of the join
  const int lp = p.splits > JOIN_FEW ? 64 : p.dh <= 32 ? 8 : p.dh <= 64 ? 16 : 32;
  const long long blocks = (rows * lp + 255) / 256;
  VITK_REQUIRE(vitk::fits_one_launch(wgs, 64 * plan.block.waves) &&
                   (p.splits == 1 || (p.splits > 64 ? vitk::fits_one_launch(rows, 64 * JOIN_WAVES) : vitk::fits_one_launch(blocks, 256))),
               "vitk_cross_sdpa_fwd: too many rows for one launch");
  hipStream_t st = vitk::as_stream(stream);
  const unsigned grid = (unsigned)wgs;
  if (plan.block.groups == 0) {
    if (p.dh <= 32)
      launch_rows<8>(p, plan.block.waves, grid, st);
    else if (p.dh <= 64)
      launch_rows<16>(p, plan.block.waves, grid, st);
    else
      launch_rows<32>(p, plan.block.waves, grid, st);
  } else if (p.dh <= 32) {
    launch_fwd<32>(p, plan.block, grid, st);
  } else if (p.dh <= 64) {
    launch_fwd<64>(p, plan.block, grid, st);
  } else if (p.dh <= 96) {
    launch_fwd<96>(p, plan.block, grid, st);
  } else {
    launch_fwd<128>(p, plan.block, grid, st);
  }
  if (p.splits > 1) {
    if (p.splits > 64)
      hipLaunchKernelGGL(cross_join_many_kernel<JOIN_WAVES>, dim3((unsigned)rows), dim3(64 * JOIN_WAVES), 0, st, p);
    else if (lp == 64)
      hipLaunchKernelGGL(cross_join_many_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    else if (lp == 8)
      hipLaunchKernelGGL(cross_join_kernel<8>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    else if (lp == 16)
      hipLaunchKernelGGL(cross_join_kernel<16>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL(cross_join_kernel<32>, dim3((unsigned)blocks), dim3(256), 0, st, p);
  }
  return vitk::check_launch("vitk_cross_sdpa_fwd");
}
