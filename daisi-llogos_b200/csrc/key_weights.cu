// What the last queries of a step give each cached key (the measure that an eviction goes by), on the CUDA cores: float32 arithmetic, storage
// float32 or bfloat16, head sizes up to 384.
//
// For sequence b of a step and key/value head h, over the rows r = (one of the last min(count, last) queries, head g of the group):
//   p_rj = e^{s_rj - M_r} / L_r over the positions j up to the query's own,  s_rj = scale q_r . k_j
//   weights[slot][h][j] = (j < len_before ? weights[slot][h][j] : 0) + sum_r p_rj
// so a key's entry starts with the step that brings the key, and rows of sequences that are not in the step are left as they were.
//
// A weight needs its row's whole sum, so there are two passes over a (sequence, head)'s keys, cut into splits: the first leaves every split's
// maximum and sum per row; the blocks of the second join those for their rows and divide.  Few rows (a decode step: the heads of a group) leave
// their scores on the way, 4 bytes a row beside a key's 2 hd bytes, and the second pass reads those; with more rows than STORE_ROWS the
// second pass works the scores out again from the keys, which then lie in L2, because storing them would be the larger traffic.
// Sums run in a fixed order everywhere.
#include "common.cuh"
#include "cache_args.h"
#include "key_weights.cuh"
#include "simt_tiles.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int THREADS = 128, ROWS = 32, MAX_HD = 384;

// A block: a split's keys of a (sequence, head), 64 at a time, ROWS rows at a time; a thread: 4 rows x 4 keys.  SECOND: the rows' ends are known.
// STAGES: tiles in shared memory, 2 where they fit: the next one's keys arrive while this one's are used.
template <typename T, bool SECOND, int STAGES>
__global__ void __launch_bounds__(THREADS) key_weights_kernel(KeyWeightArgs a) {
  constexpr int KEYS = WEIGHT_TILE, KPT = KEYS / 16;
  extern __shared__ __align__(16) float smem[];
  __shared__ float column[8][KEYS];
  __shared__ float2 ends[ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Rows s = rows_of(a, b);
  const int first = split * a.split_keys, last = min(s.total, first + a.split_keys);
  if (first >= last || s.rows <= 0) return;
  const int kp = (a.hd + 3) / 4 * 4, ks = kp + 4;
  float* Ks = smem;                        // [STAGES][KEYS][ks]
  float* Qs = Ks + STAGES * KEYS * ks;     // [ROWS][ks]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T* qg = (const T*)a.q;
  const T* kg = (const T*)a.k_pages;
  const int slot = a.slots[b], most = s.group * a.last;
  const long long pair = (long long)b * a.nkv + h;
  const TileCopy<THREADS> copy(kp);
  for (int r0 = 0; r0 < s.rows; r0 += ROWS) {
    __syncthreads();
    copy_rows<THREADS, T>(Qs, ks, ROWS, a.hd, kp, [&](int r) {
      return r0 + r < s.rows ? qg + ((long long)(s.tok0 + (r0 + r) / s.group) * a.nh + h * s.group + (r0 + r) % s.group) * a.hd : nullptr;
    });
    if (SECOND && tid < ROWS && r0 + tid < s.rows) ends[tid] = row_end(a, pair, s, r0 + tid);
    const float sc = a.scale * WEIGHT_LOG2E;
    float m[4], l[4];                      // this thread's keys alone
    int pos[4];                            // the query's own position: it sees the keys up to there
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
      pos[r] = s.pos0 + (r0 + ty * 4 + r) / s.group;
    }
    auto request = [&](int p0) {           // a tile of keys into its stage: a page's, one behind the other
      if (p0 < last)
        copy(Ks + (p0 - first) / KEYS % STAGES * KEYS * ks, ks, kg + kv_row(a.page_table, a.table_width, a.table_width, slot, p0, h, a.nkv) * a.hd, KEYS,
             s.total - p0, a.hd);
      tile_commit();
    };
    if (STAGES == 2) request(first);
    for (int p0 = first; p0 < last; p0 += KEYS) {
      __syncthreads();                     // the stage that is filled now has been read
      request(STAGES == 2 ? p0 + KEYS : p0);
      tile_wait<STAGES - 1>();
      __syncthreads();
      const float* Kt = Ks + (p0 - first) / KEYS % STAGES * KEYS * ks;
      float x[4][KPT];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < KPT; ++c) x[r][c] = 0.f;
      for (int d = 0; d < kp; d += 4) {
        float4 q[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) q[r] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + r) * ks + d);
#pragma unroll
        for (int c = 0; c < KPT; ++c) {
          const float4 k = *reinterpret_cast<const float4*>(Kt + (tx + 16 * c) * ks + d);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r][c] += q[r].x * k.x + q[r].y * k.y + q[r].z * k.z + q[r].w * k.w;
        }
      }
      float sum[KPT];
#pragma unroll
      for (int c = 0; c < KPT; ++c) sum[c] = 0.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = r0 + ty * 4 + r;
        if (row >= s.rows) continue;
        float top = m[r];
#pragma unroll
        for (int c = 0; c < KPT; ++c) {
          const int p = p0 + tx + 16 * c;
          if (p > pos[r]) x[r][c] = -INFINITY;
          if (SECOND) {
            if (p <= pos[r]) sum[c] += share(x[r][c], sc, ends[ty * 4 + r]);
          } else {
            top = fmaxf(top, ceilf(x[r][c] * sc));
            if (a.scores && p < s.total) a.scores[score_at(a, pair * most + row, p)] = x[r][c];
          }
        }
        if (!SECOND) {
          if (top != m[r]) l[r] *= whole2(m[r] - top);
          m[r] = top;
#pragma unroll
          for (int c = 0; c < KPT; ++c) l[r] += x[r][c] == -INFINITY ? 0.f : exp2f(fmaf(x[r][c], sc, -top));
        }
      }
      if (SECOND) {
#pragma unroll
        for (int c = 0; c < KPT; ++c) column[ty][tx + 16 * c] = sum[c];
        __syncthreads();
        if (tid < KEYS && p0 + tid < s.total) {
          float t = 0.f;
#pragma unroll
          for (int y = 0; y < 8; ++y) t += column[y][tid];
          add_weight(a, slot, h, p0 + tid, s.before, t, r0 > 0);
        }
      }
    }
    if (!SECOND) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float top = m[r];
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        float sum = m[r] == -INFINITY ? 0.f : l[r] * whole2(m[r] - top);
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        const int row = r0 + ty * 4 + r;
        if (row < s.rows && tx == 0) stats_of(a, pair, split)[row] = make_float2(top, sum);
      }
    }
  }
}

template <typename T, int STAGES>
int run(const KeyWeightArgs& a, cudaStream_t stream) {
  const int ks = (a.hd + 3) / 4 * 4 + 4;
  const size_t smem = sizeof(float) * (size_t)(STAGES * WEIGHT_TILE + ROWS) * ks;
  const dim3 grid(a.splits, a.nkv, a.n_seqs);
  auto go = [&](void (*kernel)(KeyWeightArgs)) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return llg_fail("key_weights: shared memory %zu: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), smem, stream, a);
    if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
    return llg_check_launch("key_weights");
  };
  if (go(key_weights_kernel<T, false, STAGES>)) return 1;
  return a.scores ? add_stored(a, stream) : go(key_weights_kernel<T, true, STAGES>);
}

}  // namespace

LLG_API int llg_key_weights_tile() { return WEIGHT_TILE; }
LLG_API int llg_key_weights_store_rows() { return STORE_ROWS; }

LLG_API int llg_key_weights_simt(const KeyWeightArgs* args, int dtype, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a)) return 1;
  LLG_REQUIRE(a.hd <= MAX_HD, "key_weights: heads of %d elements (1 to %d)", a.hd, MAX_HD);
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  if (dtype == LLG_F32) return a.hd <= 128 ? run<float, 2>(a, stream) : run<float, 1>(a, stream);
  if (dtype == LLG_BF16) return a.hd <= 128 ? run<__nv_bfloat16, 2>(a, stream) : run<__nv_bfloat16, 1>(a, stream);
  return llg_fail("key_weights: unknown dtype %d", dtype);
}
