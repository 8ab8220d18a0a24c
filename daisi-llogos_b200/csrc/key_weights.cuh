// What the two libraries that weigh keys share (key_weights.cu, key_weights_mma.cu): a sequence's rows, what blocks leave for each other, the
// pass over stored scores, and the checks.
#pragma once
#include "common.cuh"
#include "cache_args.h"

namespace {

constexpr int SIMT_KEYS = 64;       // keys per block on the CUDA cores
constexpr int STORE_ROWS = 32;      // most rows of a (sequence, head) whose scores are kept between the passes

// The rows of sequence b: its last queries' heads of one group.
struct Rows {
  int tok0, rows, group, before, total, pos0;      // first query token, rows, heads a query, cached keys, keys with the step's, first query's position
};
__device__ __forceinline__ Rows rows_of(const KeyWeightArgs& a, int b, int keys) {
  Rows s;
  const int first = a.cu_tokens[b], end = min(a.cu_tokens[b + 1], a.n_tokens), count = max(0, end - first), n = min(count, a.last);
  s.group = a.nh / a.nkv;
  s.tok0 = end - n;
  s.rows = n * s.group;
  s.before = a.len_before[b];
  s.total = min(min(s.before + count, a.weight_width), a.chunks * keys);
  s.pos0 = s.before + count - n;
  return s;
}

__device__ __forceinline__ float2 row_end(const KeyWeightArgs& a, long long row) {
  return __ldcg(reinterpret_cast<const float2*>(a.row_end) + row);
}
// e^{x - M} / L; nothing for a row whose scores are all -inf
__device__ __forceinline__ float share(float x, float2 end) { return end.x == -INFINITY ? 0.f : expf(x - end.x) * end.y; }

__device__ __forceinline__ long long score_at(const KeyWeightArgs& a, long long row, int p, int keys) { return row * a.chunks * keys + p; }

__device__ __forceinline__ void leave_stats(const KeyWeightArgs& a, long long row, int chunk, float m, float l) {
  reinterpret_cast<float2*>(a.stats)[row * a.chunks + chunk] = make_float2(m, l);
}

__device__ __forceinline__ void add_weight(const KeyWeightArgs& a, int slot, int h, int p, int before, float t) {
  float* w = a.weights + ((long long)slot * a.nkv + h) * a.weight_width + p;
  *w = (p < before ? *w : 0.f) + t;
}

// The block with the last ticket of a (sequence, head) joins the `chunks` blocks' maxima and sums per row: (M, 1 / L), a warp per row.
__device__ __forceinline__ void join_rows(const KeyWeightArgs& a, long long pair, const Rows& s, int chunks) {
  __shared__ int is_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int ticket = atomicAdd(&a.counters[pair], 1);
    is_last = ticket == chunks - 1;
    if (is_last) a.counters[pair] = 0;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long first = pair * s.group * a.last;
  for (int r = warp; r < s.rows; r += warps) {
    const float2* st = reinterpret_cast<const float2*>(a.stats) + (first + r) * a.chunks;
    float m = -INFINITY, l = 0.f;
    for (int c = lane; c < chunks; c += 32) {
      const float2 v = __ldcg(st + c);
      if (v.x == -INFINITY) continue;
      const float top = fmaxf(m, v.x);
      l = l * expf(m - top) + v.y * expf(v.x - top);
      m = top;
    }
    const float M = warp_max(m);
    l = warp_sum(m == -INFINITY ? 0.f : l * expf(m - M));
    if (lane == 0) reinterpret_cast<float2*>(a.row_end)[first + r] = make_float2(M, 1.f / l);
  }
}

// The second pass over stored scores: a thread per key.
__global__ void __launch_bounds__(256) add_stored_kernel(KeyWeightArgs a, int keys) {
  __shared__ float2 ends[STORE_ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, b = blockIdx.z;
  const Rows s = rows_of(a, b, keys);
  const long long first = ((long long)b * a.nkv + h) * s.group * a.last;
  if (threadIdx.x < s.rows) ends[threadIdx.x] = row_end(a, first + threadIdx.x);
  __syncthreads();
  const int p = blockIdx.x * 256 + threadIdx.x;
  if (p >= s.total || s.rows <= 0) return;
  float t = 0.f;
  for (int r = 0; r < s.rows; ++r) {
    const float x = __ldcg(a.scores + score_at(a, first + r, p, keys));
    t += x == -INFINITY ? 0.f : share(x, ends[r]);                 // -inf: a key behind the query
  }
  add_weight(a, a.slots[b], h, p, s.before, t);
}

inline int add_stored(const KeyWeightArgs& a, int keys, cudaStream_t stream) {
  const int most = a.chunks * keys;
  cudaError_t e = llg_launch(add_stored_kernel, dim3((most + 255) / 256, a.nkv, a.n_seqs), dim3(256), 0, stream, a, keys);
  if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("key_weights");
}

inline int check(const KeyWeightArgs& a, int keys) {
  LLG_REQUIRE(a.nh > 0 && a.nkv > 0 && a.nh % a.nkv == 0, "key_weights: %d heads are no multiple of %d key/value heads", a.nh, a.nkv);
  LLG_REQUIRE(a.hd > 0 && a.last > 0 && a.chunks > 0 && a.table_width > 0 && a.weight_width > 0, "key_weights: bad sizes");
  LLG_REQUIRE(a.nkv <= 65535 && a.n_seqs <= 65535, "key_weights: %d heads, %d sequences: more than a grid takes", a.nkv, a.n_seqs);
  LLG_REQUIRE(a.scale > 0.f, "key_weights: the softmax scale must be positive");
  LLG_REQUIRE(a.stats && a.row_end && a.counters, "key_weights: needs scratch and counters");
  LLG_REQUIRE(!a.scores || a.nh / a.nkv * a.last <= STORE_ROWS, "key_weights: %d rows' scores are not stored (at most %d)", a.nh / a.nkv * a.last,
              STORE_ROWS);
  return 0;
}

}  // namespace
