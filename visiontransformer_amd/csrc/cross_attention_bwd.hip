// Cross attention backward, three launches without atomics:
//   delta[row] = dout . out
//   dK, dV: one workgroup per 128 keys of one (batch, key head), all rows that read them in order
//   dQ:     one workgroup per 128 rows, all keys in order
// Both main kernels rebuild the probabilities from the stored row statistics,
//   p = exp2(c s - m) / l,  ds = p (dout v^T - delta),  dq = scale ds k,  dk = scale ds^T q,  dv = p^T dout,
// with products on v_mfma_f32_32x32x2_f32 arranged as in the forward: the accumulator of the first
// product is the operand of the next.
#include "cross_attention.h"

namespace {

using namespace vitk::cross;

constexpr int RB = 128;  // rows (dQ) or keys (dK, dV) per workgroup

__global__ __launch_bounds__(256) void cross_delta_kernel(const Params p) {
  const long long all = (long long)p.B * p.H * p.Nq;
  const int lane = threadIdx.x & 63;
  const long long r = blockIdx.x * 4ll + (threadIdx.x >> 6);
  if (r >= all) return;
  const long long bh = r / p.Nq, n = r % p.Nq, b = bh / p.H, h = bh % p.H;
  const float *x = p.o.ptr + (b * p.Nq + n) * p.o.ld + h * p.dh;
  const float *y = p.dout.ptr + (b * p.Nq + n) * p.dout.ld + h * p.dh;
  float s = 0.f;
  for (int d = lane; d < p.dh; d += 64) s += x[d] * y[d];
  s = vitk::wave_sum(s);
  if (lane == 0) p.delta[r] = s;
}

template <int DH>
__device__ __forceinline__ void zero(f32x16 (&x)[DH / 32]) {
#pragma unroll
  for (int n = 0; n < DH / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) x[n][i] = 0.f;
}
// columns g*DH/2 .. of one row (zeros if it does not exist)
template <int DH>
__device__ __forceinline__ void load_half(float (&f)[DH / 2], const float *row, bool ok, int g, const Params &p) {
#pragma unroll
  for (int i = 0; i < DH / 2; i += 4) {
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    if (ok) x = load_quad(row, g * (DH / 2) + i, p.dh, p.vec);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[i + e] = x[e];
  }
}
// tile [32][DH+4] of rows in LDS times the lane's half row: one 32 x 32 product
template <int DH>
__device__ __forceinline__ f32x16 product(const float *tile, const float (&f)[DH / 2], int c, int g) {
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
  for (int i = 0; i < DH / 2; i += 4) {
    const f32x4 x = *reinterpret_cast<const f32x4 *>(tile + c * (DH + 4) + g * (DH / 2) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], f[i + e], s, 0, 0, 0);
  }
  return s;
}
// acc^T[d][col] += tile^T[d][r] x[r][col]
template <int DH>
__device__ __forceinline__ void accumulate(f32x16 (&acc)[DH / 32], const float *tile, const f32x16 &x, int c, int g) {
#pragma unroll
  for (int n = 0; n < DH / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      acc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(tile[(8 * (i / 4) + 4 * g + i % 4) * (DH + 4) + 32 * n + c], x[i],
                                                    acc[n], 0, 0, 0);
}
template <int DH>
__device__ __forceinline__ void store(float *row, const f32x16 (&acc)[DH / 32], float f, int g, const Params &p) {
#pragma unroll
  for (int n = 0; n < DH / 32; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[n][4 * j + e] * f;
      store_quad(row, 32 * n + 8 * j + 4 * g, p.dh, p.vec, x);
    }
}

template <int DH>
__global__ __launch_bounds__(256) void cross_dkv_kernel(const Params p) {
  constexpr int LP = DH + 4;
  __shared__ __attribute__((aligned(16))) float qt[32 * LP], gt[32 * LP];
  __shared__ float rm[32], rl[32], rd[32];
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5, wave = threadIdx.x >> 6;
  long long wg = blockIdx.x;
  const int kb = (int)(wg % p.blocks);
  wg /= p.blocks;
  const int hk = (int)(wg % p.Hkv), b = (int)(wg / p.Hkv);
  const int len = valid_keys(p, b), key = kb * RB + wave * 32 + c;
  const bool key_ok = key < len;
  float kf[DH / 2], vf[DH / 2];
  load_half<DH>(kf, p.k.ptr + key_offset(p, p.k.ld, b, hk, key), key_ok, g, p);
  load_half<DH>(vf, p.v.ptr + key_offset(p, p.v.ld, b, hk, key), key_ok, g, p);
  f32x16 dk[DH / 32], dv[DH / 32];
  zero<DH>(dk), zero<DH>(dv);
  const int rows = kb * RB < len ? p.rows : 0;  // a block behind the length has nothing to add
  for (int t = 0; t < rows; t += 32) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < DH / 32; ++u) {
      const int quad = threadIdx.x + 256 * u, r = quad / (DH / 4), d = 4 * (quad % (DH / 4));
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
      if (t + r < rows) {
        x = load_quad(p.q.ptr + row_offset(p, p.q.ld, b, hk, t + r), d, p.dh, p.vec);
        y = load_quad(p.dout.ptr + row_offset(p, p.dout.ld, b, hk, t + r), d, p.dh, p.vec);
      }
      *reinterpret_cast<f32x4 *>(qt + r * LP + d) = x;
      *reinterpret_cast<f32x4 *>(gt + r * LP + d) = y;
    }
    if (threadIdx.x < 32) {
      const int r = t + threadIdx.x;
      float m = 0.f, f = 0.f, d = 0.f;
      if (r < rows) {
        const long long st = row_stat(p, b, hk, r);
        m = p.stats[2 * st];
        const float l = p.stats[2 * st + 1];
        f = l == 0.f ? 0.f : 1.f / l;
        d = p.delta[st];
      }
      rm[threadIdx.x] = m, rl[threadIdx.x] = f, rd[threadIdx.x] = d;
    }
    __syncthreads();
    f32x16 s = product<DH>(qt, kf, c, g), ds = product<DH>(gt, vf, c, g);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 8 * (i / 4) + 4 * g + i % 4;
      const float e = key_ok && t + r < rows ? __builtin_amdgcn_exp2f(s[i] * p.c - rm[r]) * rl[r] : 0.f;
      s[i] = e;
      ds[i] = e * (ds[i] - rd[r]);
    }
    accumulate<DH>(dv, gt, s, c, g);
    accumulate<DH>(dk, qt, ds, c, g);
  }
  if (key < p.Nk) {
    store<DH>(p.dk.ptr + key_offset(p, p.dk.ld, b, hk, key), dk, p.scale, g, p);
    store<DH>(p.dv.ptr + key_offset(p, p.dv.ld, b, hk, key), dv, 1.f, g, p);
  }
}

template <int DH>
__global__ __launch_bounds__(256) void cross_dq_kernel(const Params p) {
  constexpr int LP = DH + 4;
  __shared__ __attribute__((aligned(16))) float kt[32 * LP], vt[32 * LP];
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5, wave = threadIdx.x >> 6;
  long long wg = blockIdx.x;
  const int rb = (int)(wg % p.blocks);
  wg /= p.blocks;
  const int hk = (int)(wg % p.Hkv), b = (int)(wg / p.Hkv);
  const int len = valid_keys(p, b), row = rb * RB + wave * 32 + c;
  const bool row_ok = row < p.rows;
  float qf[DH / 2], gf[DH / 2];
  load_half<DH>(qf, p.q.ptr + row_offset(p, p.q.ld, b, hk, row_ok ? row : 0), row_ok, g, p);
  load_half<DH>(gf, p.dout.ptr + row_offset(p, p.dout.ld, b, hk, row_ok ? row : 0), row_ok, g, p);
  float m = 0.f, f = 0.f, delta = 0.f;
  if (row_ok) {
    const long long st = row_stat(p, b, hk, row);
    m = p.stats[2 * st];
    const float l = p.stats[2 * st + 1];
    f = l == 0.f ? 0.f : 1.f / l;
    delta = p.delta[st];
  }
  f32x16 dq[DH / 32];
  zero<DH>(dq);
  for (int t = 0; t < len; t += 32) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < DH / 32; ++u) {
      const int quad = threadIdx.x + 256 * u, key = quad / (DH / 4), d = 4 * (quad % (DH / 4));
      f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
      if (t + key < len) {
        x = load_quad(p.k.ptr + key_offset(p, p.k.ld, b, hk, t + key), d, p.dh, p.vec);
        y = load_quad(p.v.ptr + key_offset(p, p.v.ld, b, hk, t + key), d, p.dh, p.vec);
      }
      *reinterpret_cast<f32x4 *>(kt + key * LP + d) = x;
      *reinterpret_cast<f32x4 *>(vt + key * LP + d) = y;
    }
    __syncthreads();
    const f32x16 s = product<DH>(kt, qf, c, g);
    f32x16 ds = product<DH>(vt, gf, c, g);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = t + 8 * (i / 4) + 4 * g + i % 4;
      ds[i] = key < len ? __builtin_amdgcn_exp2f(s[i] * p.c - m) * f * (ds[i] - delta) : 0.f;
    }
    accumulate<DH>(dq, kt, ds, c, g);
  }
  if (row_ok) store<DH>(p.dq.ptr + row_offset(p, p.dq.ld, b, hk, row), dq, p.scale, g, p);
}

template <int DH>
int launch(Params p, hipStream_t st) {
  const long long heads = (long long)p.B * p.Hkv, all = (long long)p.B * p.H * p.Nq;
  const long long qb = (p.rows + RB - 1) / RB, kb = (p.Nk + RB - 1) / RB;
  VITK_REQUIRE((all + 3) / 4 < (1ll << 31) && heads * qb < (1ll << 31) && heads * kb < (1ll << 31),
               "vitk_cross_sdpa_bwd: too many rows for one launch");
  if (all) hipLaunchKernelGGL(cross_delta_kernel, dim3((unsigned)((all + 3) / 4)), dim3(256), 0, st, p);
  if (kb) {
    p.blocks = (int)kb;
    hipLaunchKernelGGL(cross_dkv_kernel<DH>, dim3((unsigned)(heads * kb)), dim3(256), 0, st, p);
  }
  if (qb) {
    p.blocks = (int)qb;
    hipLaunchKernelGGL(cross_dq_kernel<DH>, dim3((unsigned)(heads * qb)), dim3(256), 0, st, p);
  }
  return vitk::check_launch("vitk_cross_sdpa_bwd");
}

}  // namespace

extern "C" size_t vitk_cross_sdpa_bwd_workspace_bytes(const vitk_cross_sdpa_args *a) {
  if (!a || a->B <= 0 || a->H <= 0 || a->Nq <= 0) return 0;
  return (size_t)a->B * a->H * a->Nq * sizeof(float);
}

extern "C" int vitk_cross_sdpa_bwd(const vitk_cross_sdpa_args *a, vitk_stream_t stream) {
  Params p = {};
  if (check_args("vitk_cross_sdpa_bwd", a, true, &p)) return 1;
  if (p.B == 0 || (p.Nq == 0 && p.Nk == 0)) return 0;
  const size_t need = vitk_cross_sdpa_bwd_workspace_bytes(a);
  VITK_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need),
               "vitk_cross_sdpa_bwd: workspace of %zu bytes needed, %zu given", need, a->workspace ? a->workspace_bytes : 0);
  VITK_REQUIRE(need == 0 || vitk::aligned16(a->workspace), "vitk_cross_sdpa_bwd: workspace is not 16-byte aligned");
  p.delta = a->workspace;
  p.splits = 1;
  hipStream_t st = vitk::as_stream(stream);
  if (p.dh <= 32) return launch<32>(p, st);
  if (p.dh <= 64) return launch<64>(p, st);
  if (p.dh <= 96) return launch<96>(p, st);
  return launch<128>(p, st);
}
