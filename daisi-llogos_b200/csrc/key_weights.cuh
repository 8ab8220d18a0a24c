// What the two libraries that weigh keys share (key_weights.cu, key_weights_mma.cu): a sequence's rows, what blocks leave for each other, the
// pass over stored scores, and the checks.
#pragma once
#include "common.cuh"
#include "cache_args.h"

namespace {

constexpr int WEIGHT_TILE = 64;     // keys of a tile (a page); a split is a whole number of them
// Most rows of a (sequence, head) whose scores the matrix instructions' kernels keep between the passes; more go to tcgen05 where it takes the head size.
// us kept / worked out twice on mma.sync / tcgen05, 32 heads in groups of four, 8 x 8,190 keys, 8 x 500..8,190, 4 x 2,199..6,454: heads of 64, 16 rows
// 37 / 47 / 61, 20 / 27 / 38, 16 / 17 / 20; 24 rows 48 / 48 / 61, 25 / 28 / 38, 19 / 17 / 20; 32 rows 57 / 49 / 53, 29 / 28 / 33, 22 / 18 / 18; 40 rows
// - / 85 / 69, - / - / 43, - / 37 / 22.  Heads of 128, 16 rows 48 / 68 / 72, 24 / 35 / 41, 19 / 20 / 21; 24 rows 58 / 70 / 72, 30 / 36 / 42, 22 / 22 / 22;
// 32 rows 67 / 72 / 64, 35 / 37 / 36, 25 / 23 / 20; 40 rows - / 127 / 78, - / - / 45, - / 51 / 23.  (32 rows of heads of 64 would be a fifth faster
// worked out twice: their scores are as many bytes as the keys.)
constexpr int STORE_ROWS = 32;

// The rows of sequence b: its last queries' heads of one group.
struct Rows {
  int tok0, rows, group, before, total, pos0;      // first query token, rows, heads a query, cached keys, keys with the step's, first query's position
};
__device__ __forceinline__ Rows rows_of(const KeyWeightArgs& a, int b) {
  Rows s;
  const int first = a.cu_tokens[b], end = min(a.cu_tokens[b + 1], a.n_tokens), count = max(0, end - first), n = min(count, a.last);
  s.group = a.nh / a.nkv;
  s.tok0 = end - n;
  s.rows = n * s.group;
  s.before = a.len_before[b];
  s.total = min(min(s.before + count, a.weight_width), min(a.splits * a.split_keys, a.table_width * WEIGHT_TILE));      // (no key behind what holds it)
  s.pos0 = s.before + count - n;
  return s;
}

// A row's maximum M is kept in the exponent's own unit (score * scale * log2 e) and rounded up to a whole number: rescaling by 2^(M - M') is exact,
// and a share 2^(x scale log2 e - M) / L has no rounding but its own.
__device__ __forceinline__ float whole2(float d) { return d < -126.f ? 0.f : __int_as_float((127 + (int)d) << 23); }      // 2^d, d <= 0 whole or -inf
// x: a score without the scale; sc = scale * log2 e.  Nothing for a row whose scores are all -inf.
__device__ __forceinline__ float share(float x, float sc, float2 end) { return end.x == -INFINITY ? 0.f : exp2f(fmaf(x, sc, -end.x)) * end.y; }
constexpr float WEIGHT_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ long long score_at(const KeyWeightArgs& a, long long row, int p) { return row * a.splits * a.split_keys + p; }

__device__ __forceinline__ float2* stats_of(const KeyWeightArgs& a, long long pair, int split) {
  return reinterpret_cast<float2*>(a.stats) + (pair * a.splits + split) * (a.nh / a.nkv * a.last);
}

// A row's end, (M, 1 / L), from the splits' maxima and sums.
__device__ __forceinline__ float2 row_end(const KeyWeightArgs& a, long long pair, const Rows& s, int row) {
  const int n = (s.total + a.split_keys - 1) / a.split_keys, most = a.nh / a.nkv * a.last;
  const float2* st = stats_of(a, pair, 0) + row;
  float m = -INFINITY, l = 0.f;
  for (int c0 = 0; c0 < n; c0 += 8) {
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c0 + k < n ? __ldcg(st + (long long)(c0 + k) * most) : make_float2(-INFINITY, 0.f);
    float top = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, v[k].x);
    if (m != -INFINITY) l *= whole2(m - top);
#pragma unroll
    for (int k = 0; k < 8; ++k) l += v[k].x == -INFINITY ? v[k].y : v[k].y * whole2(v[k].x - top);      // (without a maximum the sum is 0, or no number)
    m = top;
  }
  return make_float2(l != l && m == -INFINITY ? 0.f : m, 1.f / l);      // scores that are no numbers: the row has to show it
}

// `again`: an earlier block of rows has written the key's entry in this launch already.
__device__ __forceinline__ void add_weight(const KeyWeightArgs& a, int slot, int h, int p, int before, float t, bool again = false) {
  float* w = a.weights + ((long long)slot * a.nkv + h) * a.weight_width + p;
  *w = (again || p < before ? *w : 0.f) + t;
}

// The second pass over stored scores: a thread takes four keys, a block's width apart, and DEEP rows of them at a time, four where there are no more;
// the first rows' scores and the keys' entries are under way while the rows' ends are worked out.  (A thread per key: twice as many blocks as run
// at once, each a chain of reads; eight sequences of 8,190 keys, 4 rows, 13 us of a call's 40, now 6 of 33.)
constexpr int ADD_THREADS = 256, ADD_KEYS = 4;
template <int DEEP>
__global__ void __launch_bounds__(ADD_THREADS) add_stored_kernel(KeyWeightArgs a) {
  constexpr int AT_ONCE = 32;                           // rows whose ends are worked out at once
  __shared__ float2 ends[AT_ONCE];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z, p0 = blockIdx.x * (ADD_THREADS * ADD_KEYS) + threadIdx.x;
  const Rows s = rows_of(a, b);
  const int slot = a.slots[b];
  if (p0 - (int)threadIdx.x >= s.total || s.rows <= 0) return;
  const long long pair = (long long)b * a.nkv + h, first = pair * s.group * a.last;
  float* w = a.weights + ((long long)slot * a.nkv + h) * a.weight_width;
  const float sc = a.scale * WEIGHT_LOG2E;
  float x[DEEP][ADD_KEYS], sum[ADD_KEYS], held[ADD_KEYS];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int r = 0; r < DEEP; ++r)
#pragma unroll
      for (int k = 0; k < ADD_KEYS; ++k) {
        const int p = p0 + k * ADD_THREADS;
        x[r][k] = r0 + r < s.rows && p < s.total ? __ldcg(a.scores + score_at(a, first + r0 + r, p)) : -INFINITY;
      }
  };
  fetch(0);
#pragma unroll
  for (int k = 0; k < ADD_KEYS; ++k) {
    const int p = p0 + k * ADD_THREADS;
    held[k] = p < s.before && p < s.total ? w[p] : 0.f;
    sum[k] = 0.f;
  }
  for (int r0 = 0; r0 < s.rows; r0 += DEEP) {
    if (r0 % AT_ONCE == 0) {
      __syncthreads();                                  // the rows before have been read
      if (threadIdx.x < AT_ONCE && r0 + (int)threadIdx.x < s.rows) ends[threadIdx.x] = row_end(a, pair, s, r0 + threadIdx.x);
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < DEEP; ++r) {
      const float2 end = ends[min(r0 + r, s.rows - 1) % AT_ONCE];
#pragma unroll
      for (int k = 0; k < ADD_KEYS; ++k) sum[k] += x[r][k] == -INFINITY ? 0.f : share(x[r][k], sc, end);       // -inf: a key behind the query
    }
    if (r0 + DEEP < s.rows) fetch(r0 + DEEP);
  }
#pragma unroll
  for (int k = 0; k < ADD_KEYS; ++k)
    if (p0 + k * ADD_THREADS < s.total) w[p0 + k * ADD_THREADS] = held[k] + sum[k];
}

inline int add_stored(const KeyWeightArgs& a, cudaStream_t stream) {
  const long long most = (long long)a.splits * a.split_keys;
  const dim3 grid((unsigned)((most + ADD_THREADS * ADD_KEYS - 1) / (ADD_THREADS * ADD_KEYS)), a.nkv, a.n_seqs);
  auto kernel = a.nh / a.nkv * a.last <= 4 ? add_stored_kernel<4> : add_stored_kernel<8>;      // (rows asked for at once)
  cudaError_t e = llg_launch(kernel, grid, dim3(ADD_THREADS), 0, stream, a);
  if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("key_weights");
}

inline int check(const KeyWeightArgs& a) {
  LLG_REQUIRE(a.nh > 0 && a.nkv > 0 && a.nh % a.nkv == 0, "key_weights: %d heads are no multiple of %d key/value heads", a.nh, a.nkv);
  LLG_REQUIRE(a.hd > 0 && a.last > 0 && a.table_width > 0 && a.weight_width > 0, "key_weights: bad sizes");
  LLG_REQUIRE(a.splits > 0 && a.split_keys > 0 && a.split_keys % WEIGHT_TILE == 0 && (long long)a.splits * a.split_keys < 2147483647LL,
              "key_weights: %d splits of %d keys", a.splits, a.split_keys);
  LLG_REQUIRE(a.nkv <= 65535 && a.n_seqs <= 65535, "key_weights: %d heads, %d sequences: more than a grid takes", a.nkv, a.n_seqs);
  LLG_REQUIRE(a.scale > 0.f, "key_weights: the softmax scale must be positive");
  LLG_REQUIRE(a.stats, "key_weights: needs scratch");
  return 0;
}

}  // namespace
