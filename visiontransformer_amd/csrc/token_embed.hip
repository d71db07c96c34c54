// Token embedding with scaling, and its gradient by sorted tokens.
//   forward:  out[i] = scale * table[index[i]]
//   backward: dtable[t] (+)= scale * sum of dout[i] over the tokens i with index[i] == t
//
// Both are bound by memory.  The backward reads dout once and writes the table once; what decides is
// that a few tokens make up most of a batch, so the work is cut by tokens, not by table rows:
//   1. a stable sort of (token, position).  Up to 8192 tokens by counting the smaller ones, one launch; more by
//      digits of 8 bits: counts per block and digit, then the scatter.  The launches also clear the table: the
//      clearing is most of their traffic and hides the latency of the sort;
//   2. sums over chunks of 32 sorted positions.  A token that lies inside one chunk is finished; one
//      that crosses a border leaves partial rows (at most one at each end of a chunk), which are
//      again a sorted list, 1/16 as long, summed the same way in chunks of 64 until at most
//      1024 chunks are left, whose parts are joined run by run.
// 32768 tokens x 768 over 32000 rows (0.20 GB): 55 us = 3.6 TB/s, of which the two sort passes with the clearing
// take 33, the sums 18 and the join 4; looking through all tokens per table row took 2444.
// Every sum has a fixed order (positions, then chunks); integer counts are the only atomics, in LDS.
#include "common.h"

#include <algorithm>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr int TPB = 256;

template <int W>
struct Cols {
  float x[W];
};
template <int W>
__device__ __forceinline__ Cols<W> load_cols(const float *p) {
  Cols<W> r;
  if constexpr (W == 4) {
    const f32x4 v = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) r.x[e] = v[e];
  } else {
    r.x[0] = *p;
  }
  return r;
}
template <int W>
__device__ __forceinline__ void store_cols(float *p, const Cols<W> &r) {
  if constexpr (W == 4)
    *reinterpret_cast<f32x4 *>(p) = f32x4{r.x[0], r.x[1], r.x[2], r.x[3]};
  else
    *p = r.x[0];
}

template <int W>
__device__ __forceinline__ void stream_cols(float *p, const Cols<W> &r) {
  if constexpr (W == 4)
    __builtin_nontemporal_store(f32x4{r.x[0], r.x[1], r.x[2], r.x[3]}, reinterpret_cast<f32x4 *>(p));
  else
    __builtin_nontemporal_store(r.x[0], p);
}

// A thread per W columns, 8 rows per workgroup: their indices are uniform, their loads all in flight.
// 16384 x 768: 11 us = 5.7 TB/s on the rows written and the table rows read once.
constexpr int ROWS = 8;
template <int W>
__global__ __launch_bounds__(TPB) void embedding_fwd_kernel(const float *__restrict__ table, long long V,
                                                            const int32_t *__restrict__ index, long long rows,
                                                            long long D, float scale, float *__restrict__ out) {
  const long long col = ((long long)blockIdx.y * blockDim.x + threadIdx.x) * W;
  if (col >= D) return;
  const long long r0 = (long long)blockIdx.x * ROWS;
  Cols<W> x[ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const long long t = r0 + u < rows ? index[r0 + u] : -1;
    x[u] = {};
    if (t >= 0 && t < V) x[u] = load_cols<W>(table + t * D + col);
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    if (r0 + u >= rows) break;
#pragma unroll
    for (int e = 0; e < W; ++e) x[u].x[e] *= scale;
    stream_cols<W>(out + (r0 + u) * D + col, x[u]);
  }
}

// ------------------------------------------------------------------------------------------ sort
constexpr int DIGITS = 256;
constexpr int MAX_BLOCKS = 512;   // blocks of a pass; each reads the counts of all of them
constexpr int BLOCK_MIN = 1024;   // tokens a block takes at least

struct Sort {
  const int32_t *key;  // first pass: the caller's index
  const int32_t *pos;  // first pass: null (the position itself)
  int32_t *key_out, *pos_out;
  int32_t *hist;       // [blocks][DIGITS]
  int n, V, chunk, blocks, shift;
  float *fill;         // the part of the table that this launch clears
  long long fill_n;
};

__device__ __forceinline__ int token(const Sort &s, int i) {
  const int k = s.key[i];
  return !s.pos && (k < 0 || k >= s.V) ? s.V : k;  // padding sorts behind the table
}

// Workgroups behind the sort's clear the table.
__device__ __forceinline__ bool clear_part(const Sort &s) {
  if ((int)blockIdx.x < s.blocks) return false;
  const long long stride = (long long)(gridDim.x - s.blocks) * blockDim.x;
  const long long first = (long long)(blockIdx.x - s.blocks) * blockDim.x + threadIdx.x;
  // scalar stores up to the first 16-byte border, then quads, then what is left
  const long long lead = min((long long)((16 - ((uintptr_t)s.fill & 15)) & 15) / 4, s.fill_n);
  const long long quads = (s.fill_n - lead) / 4;
  f32x4 *q = reinterpret_cast<f32x4 *>(s.fill + lead);
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  for (long long i = first; i < quads; i += stride) __builtin_nontemporal_store(z, q + i);
  for (long long i = first; i < lead; i += stride) s.fill[i] = 0.f;
  for (long long i = lead + 4 * quads + first; i < s.fill_n; i += stride) s.fill[i] = 0.f;
  return true;
}

__global__ __launch_bounds__(TPB) void embedding_count_kernel(const Sort s) {
  __shared__ int count[DIGITS];
  if (clear_part(s)) return;
  count[threadIdx.x] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * s.chunk, i1 = (int)min((long long)i0 + s.chunk, (long long)s.n);
  for (int i = i0 + threadIdx.x; i < i1; i += TPB) atomicAdd(&count[(token(s, i) >> s.shift) & (DIGITS - 1)], 1);
  __syncthreads();
  s.hist[blockIdx.x * DIGITS + threadIdx.x] = count[threadIdx.x];
}

// Stable: blocks in order, inside a block a quarter of its tokens per wave, inside those 64 at a time.
// After the two barriers that give every wave its first place for each digit the waves run on their own.
__global__ __launch_bounds__(TPB) void embedding_scatter_kernel(const Sort s) {
  __shared__ int scan[DIGITS];
  __shared__ int place[TPB / 64][DIGITS];
  if (clear_part(s)) return;
  const int d = threadIdx.x, lane = d & 63, wave = d >> 6;
  const int i0 = blockIdx.x * s.chunk, i1 = (int)min((long long)i0 + s.chunk, (long long)s.n);
  const int quarter = s.chunk / (TPB / 64);  // a multiple of 64
  const int w0 = (int)min((long long)i0 + wave * (long long)quarter, (long long)i1);
  const int w1 = (int)min((long long)w0 + quarter, (long long)i1);
#pragma unroll
  for (int w = 0; w < TPB / 64; ++w) place[w][d] = 0;
  int before = 0, all = 0;  // tokens of digit d in the blocks before this one, in all blocks
#pragma unroll 8
  for (int b = 0; b < s.blocks; ++b) {
    const int c = s.hist[b * DIGITS + d];
    if (b < (int)blockIdx.x) before += c;
    all += c;
  }
  int sum = all;  // inclusive scan over the digits
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(sum, off, 64);
    if (lane >= off) sum += v;
  }
  scan[d] = sum;
  __syncthreads();
  for (int i = w0 + lane; i < w1; i += 64) atomicAdd(&place[wave][(token(s, i) >> s.shift) & (DIGITS - 1)], 1);
  int at = sum - all + before;
#pragma unroll
  for (int w = 0; w < TPB / 64; ++w)
    if (w < wave) at += scan[64 * w + 63];
  __syncthreads();
#pragma unroll
  for (int w = 0; w < TPB / 64; ++w) {
    const int c = place[w][d];
    place[w][d] = at;
    at += c;
  }
  __syncthreads();
  for (int t = w0; t < w1; t += 64) {
    const int i = t + lane;
    const bool ok = i < w1;
    const int k = ok ? token(s, i) : 0, digit = (k >> s.shift) & (DIGITS - 1);
    unsigned long long same = __ballot(ok);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const unsigned long long v = __ballot(ok && (digit >> bit & 1));
      same &= digit >> bit & 1 ? v : ~v;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int to = ok ? place[wave][digit] + rank : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (ok && rank == 0) place[wave][digit] = to + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (ok) {
      s.key_out[to] = k;
      s.pos_out[to] = s.pos ? s.pos[i] : i;
    }
  }
}

// Up to RANK_TOKENS tokens in one launch instead of two a digit (8000 tokens x 192 over 4000 rows, all launches:
// 21.8 us instead of 28; over a table of one digit up to half as many, where it takes 15.8 and digits 16): a token's place is the number of tokens before it
// in the order (token, position).  A workgroup places 32, each counted by 32 threads; all tokens are in LDS.
constexpr int RANK_TOKENS = 8192, RANK_THREADS = 1024, RANK_TILE = 32, RANK_PARTS = RANK_THREADS / RANK_TILE;
__global__ __launch_bounds__(RANK_THREADS) void embedding_rank_kernel(const Sort s) {
  __shared__ __attribute__((aligned(16))) int32_t keys[RANK_TOKENS];
  __shared__ int part[RANK_PARTS][RANK_TILE];
  if (clear_part(s)) return;
  const int size = (s.n + 4 * RANK_PARTS - 1) / (4 * RANK_PARTS) * 4;  // of a part; all of them fit `keys`
#pragma unroll
  for (int u = 0; u < RANK_TOKENS / RANK_THREADS; ++u) {
    const int i = threadIdx.x + RANK_THREADS * u, k = token(s, min(i, s.n - 1));
    keys[i] = i < s.n ? k : INT32_MAX;
  }
  __syncthreads();
  const int i0 = blockIdx.x * RANK_TILE, t = threadIdx.x % RANK_TILE, i = i0 + t, own = threadIdx.x / RANK_TILE;
  const int mine = keys[i], j0 = own * size, j1 = j0 + size;
  int count = 0;
  auto four = [&](int j) { return *reinterpret_cast<const i32x4 *>(keys + j); };
#pragma unroll 4
  for (int j = j0; j < min(j1, i0); j += 4) {  // before the tile: equal ones too
    const i32x4 k = four(j);
#pragma unroll
    for (int e = 0; e < 4; ++e) count += k[e] <= mine;
  }
  for (int j = max(j0, i0); j < min(j1, i0 + RANK_TILE); j += 4) {
    const i32x4 k = four(j);
#pragma unroll
    for (int e = 0; e < 4; ++e) count += k[e] < mine || (k[e] == mine && j + e < i);
  }
#pragma unroll 4
  for (int j = max(j0, i0 + RANK_TILE); j < j1; j += 4) {
    const i32x4 k = four(j);
#pragma unroll
    for (int e = 0; e < 4; ++e) count += k[e] < mine;
  }
  part[own][t] = count;
  __syncthreads();
  if (own > 0 || i >= s.n) return;
#pragma unroll
  for (int w = 1; w < RANK_PARTS; ++w) count += part[w][t];
  s.key_out[count] = mine;
  s.pos_out[count] = i;
}

// ------------------------------------------------------------------------------------------ sums
constexpr int CHUNK1 = 32, CHUNK2 = 64, JOIN_CHUNKS = 1024;

struct Sums {
  const int32_t *key;   // sorted
  const int32_t *pos;   // first level: row of `src` of each entry.  Later levels: null, entry e is row e if flag[e]
  const int32_t *flag;
  const float *src;
  int n, V, chunks;
  long long D;
  int32_t *part_key, *part_flag;  // [2 * chunks]: what crosses the chunk's first and last border
  float *part;                    // [2 * chunks][D]
  float *dtable;
  float scale;
  int accumulate;
};

// One workgroup per chunk and block of columns, a thread per W columns.  Keys and rows of a chunk are
// loaded once, an entry a lane, and read from there as scalars, so the rows wait for one round
// trip only, all of a chunk in flight.  The levels behind the first have few chunks: a column per
// thread there, four times the workgroups.
template <int W, int CHUNK>
__global__ __launch_bounds__(TPB) void embedding_sum_kernel(const Sums s) {
  const int chunk = blockIdx.x, lane = threadIdx.x & 63;
  const int e0 = chunk * CHUNK, count = min(CHUNK, s.n - e0);
  const long long col = ((long long)blockIdx.y * blockDim.x + threadIdx.x) * W;
  const bool mine = col < s.D;
  int my_key = s.V, my_row = -1;
  if (lane < count) {
    my_key = s.key[e0 + lane];
    my_row = s.pos ? s.pos[e0 + lane] : s.flag[e0 + lane] ? e0 + lane : -1;
    if (my_key == s.V) my_row = -1;
  }
  if (lane >= count) my_key = __builtin_amdgcn_readlane(my_key, count - 1);  // the last run, without rows
  const int before = e0 > 0 ? s.key[e0 - 1] : -1, after = e0 + count < s.n ? s.key[e0 + count] : -1;
  int cur = __builtin_amdgcn_readlane(my_key, 0);
  bool head = before == cur;  // the run began in an earlier chunk
  int any = 0, head_any = 0, tail_any = 0;
  Cols<W> acc = {};
  auto flush = [&](bool goes_on) {
    if (head || goes_on) {
      if (any && mine) store_cols<W>(s.part + (2ll * chunk + (head ? 0 : 1)) * s.D + col, acc);
      (head ? head_any : tail_any) = any;
    } else if (any && mine) {
      float *dst = s.dtable + (long long)cur * s.D + col;
#pragma unroll
      for (int e = 0; e < W; ++e) acc.x[e] *= s.scale;
      if (s.accumulate) {
        const Cols<W> old = load_cols<W>(dst);
#pragma unroll
        for (int e = 0; e < W; ++e) acc.x[e] += old.x[e];
      }
      store_cols<W>(dst, acc);
    }
  };
  Cols<W> x[CHUNK];
#pragma unroll
  for (int u = 0; u < CHUNK; ++u) {
    const int row = __builtin_amdgcn_readlane(my_row, u);  // lanes behind the count hold -1
    x[u] = {};
    if (row >= 0 && mine) x[u] = load_cols<W>(s.src + (long long)row * s.D + col);
  }
#pragma unroll
  for (int u = 0; u < CHUNK; ++u) {
    const int k = __builtin_amdgcn_readlane(my_key, u);
    if (k != cur) {
      flush(false);
      head = false, any = 0, acc = {}, cur = k;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) acc.x[w] += x[u].x[w];
    any |= __builtin_amdgcn_readlane(my_row, u) >= 0;
  }
  flush(after == cur);
  if (threadIdx.x == 0 && blockIdx.y == 0) {  // entries without a row keep the order of the keys
    s.part_key[2 * chunk] = my_key;
    s.part_key[2 * chunk + 1] = cur;
    s.part_flag[2 * chunk] = head_any;
    s.part_flag[2 * chunk + 1] = tail_any;
  }
}

// The last step: one workgroup per chunk (and 64 W columns) whose last run goes on behind it adds that run's
// parts, each wave a quarter of them in order, then the four sums in order.
template <int W>
__global__ __launch_bounds__(TPB) void embedding_join_kernel(const Sums s) {
  constexpr int WAVES = TPB / 64, U = 8;
  __shared__ Cols<W> part[WAVES][64];
  const int chunk = blockIdx.x, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (!s.part_flag[2 * chunk + 1]) return;
  const int key = s.part_key[2 * chunk + 1];
  int more = 0;  // chunks behind this one that the run reaches into: those that start with its key
  for (int c = chunk + 1;; c += 64) {
    const bool in = c + lane < s.chunks && s.part_key[2 * (c + lane)] == key;
    const int n = __popcll(__ballot(in));
    more += n;
    if (n < 64) break;
  }
  const int quarter = (more + WAVES) / WAVES;  // of 1 + more parts, rounded up
  const int i0 = min(wave * quarter, more + 1), i1 = min(i0 + quarter, more + 1);
  const long long col = ((long long)blockIdx.y * 64 + lane) * W;
  Cols<W> acc = {};
  if (col < s.D) {
    for (int i = i0; i < i1; i += U) {
      Cols<W> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = {};
        if (i + u < i1) x[u] = load_cols<W>(s.part + (2ll * (chunk + i + u) + (i + u == 0)) * s.D + col);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < W; ++e) acc.x[e] += x[u].x[e];
    }
  }
  part[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || col >= s.D) return;
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
#pragma unroll
    for (int e = 0; e < W; ++e) acc.x[e] += part[w][lane].x[e];
  float *dst = s.dtable + (long long)key * s.D + col;
  Cols<W> old = {};
  if (s.accumulate) old = load_cols<W>(dst);
#pragma unroll
  for (int e = 0; e < W; ++e) acc.x[e] = old.x[e] + acc.x[e] * s.scale;
  store_cols<W>(dst, acc);
}

// Few tokens, not too large a table: no sort (528 tokens x 192 over 1000 rows: 4 us; 1000 over 6000 and 16000
// rows 6 and 12.7, by counting 15 and 15.6).  One workgroup per table row; each wave looks through its share of the
// tokens and adds the rows of its own in their order, the waves' sums are added in order.
constexpr int DIRECT_STEPS = 4;  // of 64 tokens a wave
template <int W, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void embedding_direct_kernel(const float *__restrict__ dout,
                                                               const int32_t *__restrict__ index, int n, long long D,
                                                               float scale, int accumulate, float *__restrict__ dtable) {
  constexpr int U = 8;
  __shared__ Cols<W> part[WAVES][64];
  __shared__ int found[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x;
  unsigned long long mine[DIRECT_STEPS];
  unsigned long long any = 0;
#pragma unroll
  for (int u = 0; u < DIRECT_STEPS; ++u) {
    const int i = (wave * (DIRECT_STEPS) + u) * 64 + lane;
    mine[u] = __ballot(i < n && index[i] == t);
    any |= mine[u];
  }
  if (lane == 0) found[wave] = any != 0;
  for (long long c0 = blockIdx.y * 64ll * W; c0 < D; c0 += gridDim.y * 64ll * W) {
    const long long col = c0 + lane * W;
    Cols<W> acc = {};
#pragma unroll
    for (int u = 0; u < DIRECT_STEPS; ++u) {
      const float *src = dout + (long long)(wave * (DIRECT_STEPS) + u) * 64 * D + col;
      unsigned long long left = mine[u];
      while (left) {
        Cols<W> x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          x[j] = {};
          if (left) {
            if (col < D) x[j] = load_cols<W>(src + (long long)__builtin_ctzll(left) * D);
            left &= left - 1;
          }
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
          for (int e = 0; e < W; ++e) acc.x[e] += x[j].x[e];
      }
    }
    part[wave][lane] = acc;
    __syncthreads();
    int hit = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) hit |= found[w];
    if (wave == 0 && col < D && (hit || !accumulate)) {
      float *dst = dtable + (long long)t * D + col;
      Cols<W> r = part[0][lane];
#pragma unroll
      for (int w = 1; w < WAVES; ++w)
#pragma unroll
        for (int e = 0; e < W; ++e) r.x[e] += part[w][lane].x[e];
      Cols<W> old = {};
      if (accumulate) old = load_cols<W>(dst);
#pragma unroll
      for (int e = 0; e < W; ++e) r.x[e] = old.x[e] + r.x[e] * scale;
      store_cols<W>(dst, r);
    }
    __syncthreads();
  }
}

// Waves of the direct form, 0 = sorted.  Four for up to 1024 tokens and 16384 rows; sixteen, for up to 4096 tokens, if
// the table is small enough for a few rounds of such workgroups (2000 tokens over 89 x 768: 6.2 us, sorted 13.8; 1671 x 192:
// 10.8 and 16; 3000 x 192: 17 and 16).
int direct_waves(long long n, long long V, long long D) {
  if (n <= 64 * DIRECT_STEPS * 4 && V <= 16384) return 4;
  return n <= 64 * DIRECT_STEPS * 16 && V * ((D + 255) / 256) <= 2048 ? 16 : 0;
}

struct Plan {
  int passes, blocks, chunk;  // no passes: by rank
  int levels;
  long long chunks[8];
  // offsets in the workspace, in 4-byte units
  long long key[2], pos[2], hist, part_key[8], part_flag[8], part[8], total;
};

Plan make_plan(long long n, long long V, long long D) {
  Plan p = {};
  int bits = 1;
  while ((V >> bits) != 0) ++bits;  // V itself is the key of padding
  p.passes = (bits + 7) / 8;
  if (n <= (p.passes > 1 ? RANK_TOKENS : RANK_TOKENS / 2)) p.passes = 0;
  long long blocks = (n + BLOCK_MIN - 1) / BLOCK_MIN;
  if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
  p.chunk = (int)(((n + blocks - 1) / blocks + TPB - 1) / TPB * TPB);
  p.blocks = (int)((n + p.chunk - 1) / p.chunk);
  long long at = 0;
  auto take = [&](long long count) {
    const long long r = at;
    at += (count + 63) / 64 * 64;
    return r;
  };
  for (int i = 0; i < (p.passes > 0 ? 2 : 1); ++i) p.key[i] = take(n), p.pos[i] = take(n);
  p.hist = take(p.passes > 0 ? (long long)DIGITS * p.blocks : 0);
  long long entries = n, size = CHUNK1;
  do {
    const long long c = (entries + size - 1) / size;
    p.chunks[p.levels] = c;
    p.part_key[p.levels] = take(2 * c);
    p.part_flag[p.levels] = take(2 * c);
    p.part[p.levels] = take(c > 1 ? 2 * c * D : 0);
    ++p.levels;
    entries = 2 * c;
    size = CHUNK2;
  } while (p.chunks[p.levels - 1] > JOIN_CHUNKS);
  p.total = at;
  return p;
}

unsigned threads_for(long long threads) { return (unsigned)(threads >= TPB ? TPB : (threads + 63) / 64 * 64); }

template <int W, int CHUNK>
void launch_sums(const Sums &s, hipStream_t st) {
  long long threads = (s.D + W - 1) / W;
  const unsigned tpb = threads_for(threads);
  const dim3 grid((unsigned)s.chunks, (unsigned)((threads + tpb - 1) / tpb));
  hipLaunchKernelGGL((embedding_sum_kernel<W, CHUNK>), grid, dim3(tpb), 0, st, s);
}

bool shape_ok(int64_t rows, int64_t V, int64_t D) { return rows >= 0 && D >= 0 && V >= 0; }

// rows at most 2^31 - 2^21 so that chunk ends stay below 2^31, a column block per 64 threads and grid.y
constexpr int64_t kMaxTokens = 2145386496ll, kMaxWidth = 65535ll * 64;

}  // namespace

extern "C" int vitk_embedding_fwd(const float *table, int64_t V, const int32_t *index, int64_t rows, int64_t D,
                                  float scale, float *out, vitk_stream_t stream) {
  VITK_REQUIRE(shape_ok(rows, V, D), "vitk_embedding_fwd: bad shape");
  if (rows == 0 || D == 0) return 0;
  VITK_REQUIRE(index && out && (table || V == 0), "vitk_embedding_fwd: null pointer");
  VITK_REQUIRE(out != table, "vitk_embedding_fwd: out is the table");
  VITK_REQUIRE(V <= INT32_MAX, "vitk_embedding_fwd: table of %lld rows", (long long)V);
  const bool vec = D % 4 == 0 && vitk::aligned16(table) && vitk::aligned16(out);
  hipStream_t st = vitk::as_stream(stream);
  const long long threads = vec ? D / 4 : D, groups = (rows + ROWS - 1) / ROWS;
  const unsigned tpb = threads_for(threads);
  VITK_REQUIRE(rows <= INT64_MAX - ROWS && D <= kMaxWidth, "vitk_embedding_fwd: %lld rows of %lld", (long long)rows,
               (long long)D);
  auto kernel = vec ? embedding_fwd_kernel<4> : embedding_fwd_kernel<1>;
  const long long most = (1ll << 32) / tpb - 1;  // groups of one launch, which has fewer than 2^32 threads in a dimension
  for (long long g0 = 0; g0 < groups; g0 += most) {
    const dim3 grid((unsigned)std::min(most, groups - g0), (unsigned)((threads + tpb - 1) / tpb));
    hipLaunchKernelGGL(kernel, grid, dim3(tpb), 0, st, table, (long long)V, index + g0 * ROWS, (long long)rows - g0 * ROWS,
                       (long long)D, scale, out + g0 * ROWS * D);
  }
  return vitk::check_launch("vitk_embedding_fwd");
}

extern "C" size_t vitk_embedding_bwd_workspace_bytes(int64_t rows, int64_t V, int64_t D) {
  if (!shape_ok(rows, V, D) || rows == 0 || V == 0 || D == 0 || rows > kMaxTokens || direct_waves(rows, V, D) > 0) return 0;
  return (size_t)make_plan(rows, V, D).total * 4;
}

extern "C" int vitk_embedding_bwd(const float *dout, const int32_t *index, int64_t rows, int64_t V, int64_t D,
                                  float scale, int32_t accumulate, float *dtable, float *workspace,
                                  size_t workspace_bytes, vitk_stream_t stream) {
  VITK_REQUIRE(shape_ok(rows, V, D), "vitk_embedding_bwd: bad shape");
  if (V == 0 || D == 0) return 0;
  VITK_REQUIRE(dtable && (rows == 0 || (dout && index)), "vitk_embedding_bwd: null pointer");
  VITK_REQUIRE(dtable != dout, "vitk_embedding_bwd: dtable is dout");
  VITK_REQUIRE(V <= INT32_MAX && rows <= kMaxTokens && D <= kMaxWidth,
               "vitk_embedding_bwd: %lld tokens over a table of %lld rows of %lld", (long long)rows, (long long)V,
               (long long)D);
  hipStream_t st = vitk::as_stream(stream);
  if (rows == 0) return accumulate ? 0 : vitk_fill_f32(dtable, 0.f, V * D, stream);
  const bool vec = D % 4 == 0 && vitk::aligned16(dout) && vitk::aligned16(dtable);
  if (const int waves = direct_waves(rows, V, D)) {
    // few table rows: a workgroup for each block of their columns (756 tokens x 1024 over 51 rows: 14 -> 6 us, 1000
    // over 2000 rows 10 -> 8, over 4000 11 -> 14)
    const int width = vec ? 256 : 64;
    const long long blocks = (D + width - 1) / width;
    const dim3 grid((unsigned)V, V * blocks <= 8192 ? (unsigned)blocks : 1), block(64 * waves);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, block, 0, st, dout, index, (int)rows, (long long)D, scale, (int)accumulate, dtable);
    };
    if (waves == 4)
      vec ? launch(embedding_direct_kernel<4, 4>) : launch(embedding_direct_kernel<1, 4>);
    else
      vec ? launch(embedding_direct_kernel<4, 16>) : launch(embedding_direct_kernel<1, 16>);
    return vitk::check_launch("vitk_embedding_bwd");
  }
  const Plan p = make_plan(rows, V, D);
  VITK_REQUIRE(workspace && workspace_bytes >= (size_t)p.total * 4,
               "vitk_embedding_bwd: workspace of %zu bytes needed, %zu given", (size_t)p.total * 4,
               workspace ? workspace_bytes : 0);
  VITK_REQUIRE(vitk::aligned16(workspace), "vitk_embedding_bwd: workspace is not 16-byte aligned");
  VITK_REQUIRE(vitk::fits_one_launch(p.chunks[0], (int)threads_for(vec ? D / 4 : D)),
               "vitk_embedding_bwd: %lld tokens of %lld in one launch", (long long)rows, (long long)D);
  int32_t *iw = reinterpret_cast<int32_t *>(workspace);
  Sort s = {};
  s.n = (int)rows, s.V = (int)V, s.chunk = p.chunk, s.blocks = p.blocks, s.hist = iw + p.hist;
  // the clearing, a tenth to each count and the rest to the scatters, which take longer (multiples of 4 floats)
  const long long all = accumulate ? 0 : V * D;
  long long cleared = 0;
  auto sort_launch = [&](void (*kernel)(Sort), unsigned threads, long long share, bool last) {
    share = (share + 3) / 4 * 4;
    s.fill = dtable + cleared;
    s.fill_n = last ? all - cleared : std::min(share, all - cleared);
    cleared += s.fill_n;
    const long long want = (s.fill_n / 4 + threads * 4 - 1) / (threads * 4);
    const unsigned grid = (unsigned)(s.blocks + std::min(want, (long long)(2048 * TPB / threads)) + (s.fill_n > 0 && want == 0));
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, st, s);
  };
  if (p.passes == 0) {
    s.blocks = (int)((rows + RANK_TILE - 1) / RANK_TILE);
    s.key = index, s.key_out = iw + p.key[0], s.pos_out = iw + p.pos[0];
    sort_launch(embedding_rank_kernel, RANK_THREADS, all, true);
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    s.key = pass == 0 ? index : iw + p.key[1 - (pass & 1)];
    s.pos = pass == 0 ? nullptr : iw + p.pos[1 - (pass & 1)];
    s.key_out = iw + p.key[pass & 1], s.pos_out = iw + p.pos[pass & 1];
    s.shift = 8 * pass;
    sort_launch(embedding_count_kernel, TPB, all / p.passes / 5, false);
    sort_launch(embedding_scatter_kernel, TPB, all / p.passes * 4 / 5, pass + 1 == p.passes);
  }
  Sums q = {};
  q.key = s.key_out, q.pos = s.pos_out, q.src = dout;
  q.V = (int)V, q.D = D, q.dtable = dtable, q.scale = scale, q.accumulate = accumulate;
  long long entries = rows;
  for (int level = 0; level < p.levels; ++level) {
    q.n = (int)entries, q.chunks = (int)p.chunks[level];
    q.part_key = iw + p.part_key[level], q.part_flag = iw + p.part_flag[level], q.part = workspace + p.part[level];
    if (level > 0)
      launch_sums<1, CHUNK2>(q, st);
    else if (vec)
      launch_sums<4, CHUNK1>(q, st);
    else
      launch_sums<1, CHUNK1>(q, st);
    if (level + 1 == p.levels && p.chunks[level] > 1) {
      const unsigned width = vec ? 256 : 64;  // columns of a workgroup
      const dim3 grid((unsigned)q.chunks, (unsigned)((D + width - 1) / width));
      if (vec)
        hipLaunchKernelGGL(embedding_join_kernel<4>, grid, dim3(TPB), 0, st, q);
      else
        hipLaunchKernelGGL(embedding_join_kernel<1>, grid, dim3(TPB), 0, st, q);
    }
    q.key = q.part_key, q.flag = q.part_flag, q.src = q.part, q.pos = nullptr;
    entries = 2 * p.chunks[level];
  }
  return vitk::check_launch("vitk_embedding_bwd");
}
