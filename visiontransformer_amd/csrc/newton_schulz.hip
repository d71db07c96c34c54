// Orthogonalised updates: y = x / (|x|_F + eps), then `steps` times g = y y^T, y = a y + (b g + c g g) y,
// and the Muon step that applies the result to a parameter.
//
// The matrices are held with their shorter side (r) as rows (a taller matrix is transposed on the way in and
// out: the polynomial acts on singular values only) and padded with zeros to multiples of 64.
// Products run on v_mfma_f32_32x32x16_f16 with every fp32 operand x split in two fp16 parts,
//   2^S x = hi + lo,  hi = fp16(2^S x), lo = fp16(2^S x - hi),
// and x y = hi hi' + hi lo' + lo hi' with fp32 sums: 22 significant bits (the dropped lo lo' is below
// 2^-22), on matrix cores that do fp16 at 16 times the rate of fp32.  The steps are normalised, so
// the range is known and the scales are constants: |y| <= 4 with S = 12 (a head room of 16), |y y^T| <= 16
// and |b g + c g g| < 31 with S = 10 (head room 64).  Against 64 bits the result is as close as the
// same steps in fp32 throughout (the error is that of the long sums, not of the operands).
// The iterate itself and the norms stay in fp32 / fp64.
#include "common.h"

#include <cmath>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int T = 64;         // output tile
constexpr int KS = 32;        // contraction per slab
constexpr int LP = KS + 8;    // LDS pitch in fp16
constexpr int PARTS = 64;     // partial sums of a norm
constexpr float kY = 4096.f, kG = 1024.f;  // 2^S of the planes of y and of g, b g + c g g

struct Planes {  // hi and lo part of an fp32 matrix
  _Float16 *hi, *lo;
};

struct NsParams {
  // the user's matrices (row-major, as given)
  const float *x;      // Newton-Schulz: input.  Muon: gradient
  float *m, *p, *out;  // Muon: momentum, parameter.  Newton-Schulz: out
  long long ld_x, stride_x, ld_out, stride_out;
  int rows, cols, batch, tall;  // tall: rows > cols
  float momentum, grad_scale, keep, step;
  int nesterov;
  float a, b, c, eps;
  // workspace
  int r, n, rp, np;
  float *y, *g;                     // [batch][rp][np], [batch][rp][rp]
  Planes yp, yt[2], gp, bp;         // y, y^T ([np][rp]; read and written by one product, so two), g, b g + c g g
  double *sums;                     // [batch][PARTS]
};

__device__ __forceinline__ void split(float v, _Float16 &hi, _Float16 &lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

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

// Sum of squares of one matrix in PARTS parts, each over whole rows in a fixed order; Muon: the new momentum.
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsParams p) {
  __shared__ double red[4];
  const int part = blockIdx.x % PARTS;
  const long long k = blockIdx.x / PARTS;
  const long long size = (long long)p.rows * p.cols, chunk = (size + PARTS - 1) / PARTS;
  const long long end = (part + 1) * chunk < size ? (part + 1) * chunk : size;
  double s = 0.0;
  for (long long i = part * chunk + threadIdx.x; i < end; i += 256) {
    const long long row = i / p.cols;
    const float u = update_value(p, k * p.stride_x + row * p.ld_x + (i - row * p.cols), true);
    s += (double)u * (double)u;
  }
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
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

// y = u / (|u| + eps) with its planes and transposed planes, one 64 x 64 tile per workgroup; `last`: only the result.
__global__ __launch_bounds__(256) void ns_start_kernel(const NsParams p, int last) {
  __shared__ float tile[T][T + 1];
  const int tj = p.np / T, tiles = (p.rp / T) * tj;
  const long long k = blockIdx.x / tiles;
  const int t = blockIdx.x % tiles, i0 = t / tj * T, j0 = t % tj * T;
  double s = 0.0;
  for (int part = 0; part < PARTS; ++part) s += p.sums[k * PARTS + part];
  const float norm = (float)sqrt(s) + p.eps;
  for (int u = threadIdx.x; u < T * T; u += 256) {  // walk the user's matrix along its rows
    const int a = u / T, b = u % T, i = p.tall ? b : a, j = p.tall ? a : b;
    float v = 0.f;
    if (i0 + i < p.r && j0 + j < p.n) {
      const long long row = p.tall ? j0 + j : i0 + i, col = p.tall ? i0 + i : j0 + j;
      v = update_value(p, k * p.stride_x + row * p.ld_x + col, false) / norm;
    }
    tile[i][j] = v;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < T * T; u += 256) {
    const int i = u / T, j = u % T;
    const float v = tile[i][j];
    if (last) {
      emit(p, k, i0 + i, j0 + j, v);
      continue;
    }
    const long long at = (k * p.rp + i0 + i) * p.np + j0 + j;
    p.y[at] = v;
    split(v * kY, p.yp.hi[at], p.yp.lo[at]);
    const long long tt = (k * p.np + j0 + i) * p.rp + i0 + j;
    split(tile[j][i] * kY, p.yt[0].hi[tt], p.yt[0].lo[tt]);
  }
}

enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

// C[i][j] = sum_k P[i][k] Q[j][k], one 64 x 64 tile per workgroup, a wave per 32 x 32 quarter.
//   GRAM: P = Q = y      -> g and its planes
//   POLY: P = Q = g      -> planes of b g + c g g
//   APPLY: P = that, Q = y^T -> y = a y + C with its planes;  LAST: the same, result to the user's matrix
template <int MODE>
__global__ __launch_bounds__(256) void ns_product_kernel(const NsParams p, int flip) {
  __shared__ __attribute__((aligned(16))) _Float16 lds[2][2][T * LP];  // operand, part
  const int cols = MODE >= APPLY ? p.np : p.rp, depth = MODE == GRAM ? p.np : p.rp;
  const int tj = cols / T, tiles = (p.rp / T) * tj;
  const long long k = blockIdx.x / tiles;
  const int t = blockIdx.x % tiles, i0 = t / tj * T, j0 = t % tj * T;
  const Planes P = MODE == GRAM ? p.yp : MODE == POLY ? p.gp : p.bp;
  const Planes Q = MODE == GRAM ? p.yp : MODE == POLY ? p.gp : p.yt[flip];
  const long long pb = (k * p.rp + i0) * depth, qb = (k * (long long)cols + j0) * depth;
  const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5, wave = threadIdx.x >> 6;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 8;  // this thread's 16 bytes of a slab
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < depth; k0 += KS) {
    const long long po = pb + (long long)lr * depth + k0 + lc, qo = qb + (long long)lr * depth + k0 + lc;
    const f16x8 x0 = *reinterpret_cast<const f16x8 *>(P.hi + po), x1 = *reinterpret_cast<const f16x8 *>(P.lo + po);
    const f16x8 y0 = *reinterpret_cast<const f16x8 *>(Q.hi + qo), y1 = *reinterpret_cast<const f16x8 *>(Q.lo + qo);
    __syncthreads();
    *reinterpret_cast<f16x8 *>(&lds[0][0][lr * LP + lc]) = x0;
    *reinterpret_cast<f16x8 *>(&lds[0][1][lr * LP + lc]) = x1;
    *reinterpret_cast<f16x8 *>(&lds[1][0][lr * LP + lc]) = y0;
    *reinterpret_cast<f16x8 *>(&lds[1][1][lr * LP + lc]) = y1;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < KS; h += 16) {
      const f16x8 ph = *reinterpret_cast<const f16x8 *>(&lds[0][0][(wi + c) * LP + h + 8 * g]);
      const f16x8 pl = *reinterpret_cast<const f16x8 *>(&lds[0][1][(wi + c) * LP + h + 8 * g]);
      const f16x8 qh = *reinterpret_cast<const f16x8 *>(&lds[1][0][(wj + c) * LP + h + 8 * g]);
      const f16x8 ql = *reinterpret_cast<const f16x8 *>(&lds[1][1][(wj + c) * LP + h + 8 * g]);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    }
  }
  const int j = j0 + wj + c;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int i = i0 + wi + 8 * (e / 4) + 4 * g + e % 4;
    const long long at = (k * p.rp + i) * cols + j;
    if (MODE == GRAM) {
      const float v = acc[e] * (1.f / (kY * kY));
      p.g[at] = v;
      split(v * kG, p.gp.hi[at], p.gp.lo[at]);
    } else if (MODE == POLY) {
      const float v = p.b * p.g[at] + p.c * (acc[e] * (1.f / (kG * kG)));
      split(v * kG, p.bp.hi[at], p.bp.lo[at]);
    } else {
      const float v = p.a * p.y[at] + acc[e] * (1.f / (kG * kY));
      if (MODE == LAST) {
        emit(p, k, i, j, v);
      } else {
        p.y[at] = v;
        _Float16 hi, lo;
        split(v * kY, hi, lo);
        p.yp.hi[at] = hi, p.yp.lo[at] = lo;
        const long long tt = (k * p.np + j) * p.rp + i;
        p.yt[1 - flip].hi[tt] = hi, p.yt[1 - flip].lo[tt] = lo;
      }
    }
  }
}

long long padded(long long x) { return (x + T - 1) / T * T; }

// Workspace of one call: sums, then y, g (fp32), then the planes.
size_t plan(NsParams *p, float *workspace) {
  p->tall = p->rows > p->cols;
  p->r = p->tall ? p->cols : p->rows;
  p->n = p->tall ? p->rows : p->cols;
  p->rp = (int)padded(p->r);
  p->np = (int)padded(p->n);
  const size_t b = p->batch, yy = b * p->rp * p->np, gg = b * p->rp * p->rp;
  char *at = reinterpret_cast<char *>(workspace);
  size_t used = 0;
  auto take = [&](size_t bytes) {
    char *r = at ? at + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return r;
  };
  p->sums = reinterpret_cast<double *>(take(b * PARTS * sizeof(double)));
  p->y = reinterpret_cast<float *>(take(yy * 4));
  p->g = reinterpret_cast<float *>(take(gg * 4));
  auto planes = [&](size_t count) {
    Planes r;
    r.hi = reinterpret_cast<_Float16 *>(take(count * 2));
    r.lo = reinterpret_cast<_Float16 *>(take(count * 2));
    return r;
  };
  p->yp = planes(yy), p->yt[0] = planes(yy), p->yt[1] = planes(yy), p->gp = planes(gg), p->bp = planes(gg);
  return used;
}

bool size_ok(int64_t rows, int64_t cols, int64_t batch) {
  return rows >= 0 && cols >= 0 && batch >= 0 && rows <= (1 << 20) && cols <= (1 << 20);
}

// Does the iteration t -> a t + b t^3 + c t^5 stay where the fixed scales hold?
bool bounded(float a, float b, float c, int steps) {
  for (int i = 0; i <= 64; ++i) {
    double t = i / 64.0;
    for (int s = 0; s < steps; ++s) {
      const double q = t * t, poly = b * q + c * q * q;
      if (!(std::fabs(poly) < 31.0)) return false;
      t = a * t + poly * t;
      if (!(std::fabs(t) <= 4.0)) return false;
    }
  }
  return true;
}

int run(const char *who, NsParams *p, int steps, float *workspace, size_t bytes, hipStream_t st) {
  const size_t need = plan(p, nullptr);
  VITK_REQUIRE(workspace && bytes >= need, "%s: workspace of %zu bytes needed, %zu given", who, need,
               workspace ? bytes : 0);
  VITK_REQUIRE(vitk::aligned16(workspace), "%s: workspace is not 16-byte aligned", who);
  plan(p, workspace);
  const long long ti = p->rp / T, tj = p->np / T, yb = p->batch * ti * tj, gb = p->batch * ti * ti;
  VITK_REQUIRE(yb < (1ll << 31) && p->batch * (long long)PARTS < (1ll << 31), "%s: too many matrices for one launch", who);
  const dim3 block(256);
  hipLaunchKernelGGL(ns_norm_kernel, dim3(p->batch * PARTS), block, 0, st, *p);
  hipLaunchKernelGGL(ns_start_kernel, dim3((unsigned)yb), block, 0, st, *p, steps == 0 ? 1 : 0);
  for (int s = 0; s < steps; ++s) {
    hipLaunchKernelGGL(ns_product_kernel<GRAM>, dim3((unsigned)gb), block, 0, st, *p, 0);
    hipLaunchKernelGGL(ns_product_kernel<POLY>, dim3((unsigned)gb), block, 0, st, *p, 0);
    if (s + 1 < steps)
      hipLaunchKernelGGL(ns_product_kernel<APPLY>, dim3((unsigned)yb), block, 0, st, *p, s & 1);
    else
      hipLaunchKernelGGL(ns_product_kernel<LAST>, dim3((unsigned)yb), block, 0, st, *p, s & 1);
  }
  return vitk::check_launch(who);
}

size_t bytes_of(int32_t rows, int32_t cols, int32_t batch) {
  if (!size_ok(rows, cols, batch) || rows == 0 || cols == 0 || batch == 0) return 0;
  NsParams p = {};
  p.rows = rows, p.cols = cols, p.batch = batch;
  return plan(&p, nullptr);
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
  NsParams p = {};
  p.x = a->x, p.out = a->out;
  p.ld_x = a->ld_x, p.stride_x = a->stride_x, p.ld_out = a->ld_out, p.stride_out = a->stride_out;
  p.rows = a->rows, p.cols = a->cols, p.batch = a->batch;
  p.a = a->a, p.b = a->b, p.c = a->c, p.eps = a->eps;
  return run(who, &p, a->steps, a->workspace, a->workspace_bytes, vitk::as_stream(stream));
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
  p.rows = a->rows, p.cols = a->cols, p.batch = a->batch;
  p.momentum = a->momentum, p.grad_scale = a->grad_scale, p.nesterov = a->nesterov;
  p.keep = 1.f - a->lr * a->weight_decay, p.step = a->lr * a->update_scale;
  p.a = a->a, p.b = a->b, p.c = a->c, p.eps = a->eps;
  return run(who, &p, a->steps, a->workspace, a->workspace_bytes, vitk::as_stream(stream));
}
