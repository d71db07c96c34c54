// Token embedding with scaling, and its gradient.
//   forward:  out[i] = scale * table[index[i]]
//   backward: dtable[t] (+)= scale * sum of dout[i] over the tokens i with index[i] == t, in token order
#include "common.h"

#include <cmath>

namespace {

constexpr int TPB = 256;

__global__ __launch_bounds__(TPB) void embedding_fwd_kernel(const float *__restrict__ table, long long V,
                                                            const int32_t *__restrict__ index, long long rows,
                                                            long long D, float scale, float *__restrict__ out) {
  const long long total = rows * D;
  for (long long i = blockIdx.x * (long long)TPB + threadIdx.x; i < total; i += (long long)gridDim.x * TPB) {
    const long long r = i / D, c = i - r * D;
    const long long t = index[r];
    out[i] = t >= 0 && t < V ? scale * table[t * D + c] : 0.f;
  }
}

// One workgroup per row of the table: it looks through all tokens, 256 at a time, and adds the rows
// of its own in their order.
__global__ __launch_bounds__(TPB) void embedding_bwd_kernel(const float *__restrict__ dout,
                                                            const int32_t *__restrict__ index, long long rows,
                                                            long long V, long long D, float scale, int accumulate,
                                                            float *__restrict__ dtable) {
  __shared__ int found[TPB];
  __shared__ int count[TPB / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (long long t = blockIdx.x; t < V; t += gridDim.x) {
    for (long long c0 = 0; c0 < D; c0 += TPB) {
      const long long c = c0 + threadIdx.x;
      float sum = 0.f;
      int any = 0;
      for (long long i0 = 0; i0 < rows; i0 += TPB) {
        const long long i = i0 + threadIdx.x;
        const bool mine = i < rows && index[i] == t;
        const unsigned long long votes = __ballot(mine);
        __syncthreads();  // found may still be read
        if (lane == 0) count[wave] = __popcll(votes);
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < TPB / 64; ++w) {
          if (w < wave) before += count[w];
          all += count[w];
        }
        if (mine) found[before + __popcll(votes & ((1ull << lane) - 1))] = threadIdx.x;
        __syncthreads();
        if (c < D)
          for (int j = 0; j < all; ++j) sum += dout[(i0 + found[j]) * D + c];
        any += all;
      }
      if (c < D) {
        float *dst = dtable + t * D + c;
        if (accumulate) {
          if (any) *dst += scale * sum;
        } else {
          *dst = scale * sum;
        }
      }
    }
  }
}

}  // namespace

extern "C" int vitk_embedding_fwd(const float *table, int64_t V, const int32_t *index, int64_t rows, int64_t D,
                                  float scale, float *out, vitk_stream_t stream) {
  VITK_REQUIRE(rows >= 0 && D >= 0 && V >= 0, "vitk_embedding_fwd: bad shape");
  if (rows == 0 || D == 0) return 0;
  VITK_REQUIRE(index && out && (table || V == 0), "vitk_embedding_fwd: null pointer");
  VITK_REQUIRE(V <= INT32_MAX, "vitk_embedding_fwd: table of %lld rows", (long long)V);
  hipLaunchKernelGGL(embedding_fwd_kernel, dim3(vitk::grid_for(rows * D, TPB)), dim3(TPB), 0, vitk::as_stream(stream),
                     table, (long long)V, index, (long long)rows, (long long)D, scale, out);
  return vitk::check_launch("vitk_embedding_fwd");
}

extern "C" size_t vitk_embedding_bwd_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int vitk_embedding_bwd(const float *dout, const int32_t *index, int64_t rows, int64_t V, int64_t D,
                                  float scale, int32_t accumulate, float *dtable, float *, size_t,
                                  vitk_stream_t stream) {
  VITK_REQUIRE(rows >= 0 && D >= 0 && V >= 0, "vitk_embedding_bwd: bad shape");
  if (V == 0 || D == 0) return 0;
  VITK_REQUIRE(dtable && (rows == 0 || (dout && index)), "vitk_embedding_bwd: null pointer");
  VITK_REQUIRE(V <= INT32_MAX && rows <= INT32_MAX, "vitk_embedding_bwd: %lld tokens over a table of %lld rows",
               (long long)rows, (long long)V);
  const unsigned blocks = (unsigned)(V < 65536 ? V : 65536);
  hipLaunchKernelGGL(embedding_bwd_kernel, dim3(blocks), dim3(TPB), 0, vitk::as_stream(stream), dout, index,
                     (long long)rows, (long long)V, (long long)D, scale, (int)accumulate, dtable);
  return vitk::check_launch("vitk_embedding_bwd");
}
