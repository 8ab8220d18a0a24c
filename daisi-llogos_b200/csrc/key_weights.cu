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
// their scores on the way, 4 bytes a row beside a key's 2 hd bytes, and the second pass reads those; on the matrix instructions with more rows than
// STORE_ROWS, and everywhere where the scores would be more than a workspace should be, the second pass works them out again from the keys.
// Sums run in a fixed order everywhere.
//
// What bounds it: reads of shared memory for the products, and for small calls the two passes' latency.  float32, us with scores kept / worked out
// twice: a decode step of 8 x 4,000 keys, 32 heads of 128 in groups of four, 60 / 120 (the keys alone 21); 13 x 1,106, 38 / 73; 32 queries of two
// prompts of 2,000 to 4,000, 105 / 205; 17 queries of five of 748, 9 heads of 48, 23 / 34.  (With 32 rows to a block whatever their number, row blocks
// one after the other, one product an instruction and splits of four tiles: 130, 75, 283 and 59.)
#include "common.cuh"
#include "cache_args.h"
#include "key_weights.cuh"
#include "simt_tiles.cuh"

#include <algorithm>

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int THREADS = 128, MAX_HD = 384;

// A block: a split's keys of a (sequence, head), 64 at a time, and 8 RY rows, or in the second pass all rows, 8 RY at a time; a thread: RY rows x 4
// keys, two products an instruction.  SECOND: the rows' ends are known.  STAGES: tiles in shared memory, 2 where they fit: the next one's keys
// arrive while this one's are used.
template <typename T, int RY, bool SECOND, int STAGES>
__global__ void __launch_bounds__(THREADS) key_weights_kernel(KeyWeightArgs a) {
  constexpr int KEYS = WEIGHT_TILE, KPT = KEYS / 16, ROWS = 8 * RY;
  extern __shared__ __align__(16) float smem[];
  __shared__ float column[8][KEYS];
  __shared__ float2 ends[ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int row_blocks = gridDim.y / a.nkv, split = blockIdx.x, h = blockIdx.y / row_blocks, b = blockIdx.z;
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
  for (int r0 = ((int)blockIdx.y - h * row_blocks) * ROWS; r0 < s.rows; r0 += row_blocks * ROWS) {
    __syncthreads();
    copy_rows<THREADS, T>(Qs, ks, ROWS, a.hd, kp, [&](int r) {
      return r0 + r < s.rows ? qg + ((long long)(s.tok0 + (r0 + r) / s.group) * a.nh + h * s.group + (r0 + r) % s.group) * a.hd : nullptr;
    });
    if (SECOND && tid < ROWS && r0 + tid < s.rows) ends[tid] = row_end(a, pair, s, r0 + tid);
    const float sc = a.scale * WEIGHT_LOG2E;
    float m[RY], l[RY];                    // this thread's keys alone
    int pos[RY];                           // the query's own position: it sees the keys up to there
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
      pos[r] = s.pos0 + (r0 + ty * RY + r) / s.group;
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
      float2 x2[RY][KPT];                  // elements 0, 2, ... and 1, 3, ...
#pragma unroll
      for (int r = 0; r < RY; ++r)
#pragma unroll
        for (int c = 0; c < KPT; ++c) x2[r][c] = make_float2(0.f, 0.f);
#pragma unroll 2
      for (int d = 0; d < kp; d += 4) {
        float4 q[RY];
#pragma unroll
        for (int r = 0; r < RY; ++r) q[r] = *reinterpret_cast<const float4*>(Qs + (ty * RY + r) * ks + d);
#pragma unroll
        for (int c = 0; c < KPT; ++c) {
          const float4 k = *reinterpret_cast<const float4*>(Kt + (tx + 16 * c) * ks + d);
#pragma unroll
          for (int r = 0; r < RY; ++r) {
            x2[r][c] = __ffma2_rn(make_float2(q[r].x, q[r].y), make_float2(k.x, k.y), x2[r][c]);
            x2[r][c] = __ffma2_rn(make_float2(q[r].z, q[r].w), make_float2(k.z, k.w), x2[r][c]);
          }
        }
      }
      float x[RY][KPT];
#pragma unroll
      for (int r = 0; r < RY; ++r)
#pragma unroll
        for (int c = 0; c < KPT; ++c) x[r][c] = x2[r][c].x + x2[r][c].y;
      float sum[KPT];
#pragma unroll
      for (int c = 0; c < KPT; ++c) sum[c] = 0.f;
#pragma unroll
      for (int r = 0; r < RY; ++r) {
        const int row = r0 + ty * RY + r;
        if (row >= s.rows) continue;
        float top = m[r];
#pragma unroll
        for (int c = 0; c < KPT; ++c) {
          const int p = p0 + tx + 16 * c;
          if (p > pos[r]) x[r][c] = -INFINITY;
          if (SECOND) {
            if (p <= pos[r]) sum[c] += share(x[r][c], sc, ends[ty * RY + r]);
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
      for (int r = 0; r < RY; ++r) {
        float top = m[r];
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        float sum = m[r] == -INFINITY ? l[r] : l[r] * whole2(m[r] - top);
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        const int row = r0 + ty * RY + r;
        if (row < s.rows && tx == 0) stats_of(a, pair, split)[row] = make_float2(top, sum);
      }
    }
  }
}

template <typename T, int RY, int STAGES>
int run(const KeyWeightArgs& a, cudaStream_t stream) {
  const int ks = (a.hd + 3) / 4 * 4 + 4;
  const size_t smem = sizeof(float) * (size_t)(STAGES * WEIGHT_TILE + 8 * RY) * ks;
  const int rows = a.nh / a.nkv * a.last, row_blocks = std::min((rows + 8 * RY - 1) / (8 * RY), 65535 / a.nkv);
  auto go = [&](void (*kernel)(KeyWeightArgs), int rbs) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return llg_fail("key_weights: shared memory %zu: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, dim3(a.splits, a.nkv * rbs, a.n_seqs), dim3(THREADS), smem, stream, a);
    if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
    return llg_check_launch("key_weights");
  };
  if (go(key_weights_kernel<T, RY, false, STAGES>, row_blocks)) return 1;
  return a.scores ? add_stored(a, stream) : go(key_weights_kernel<T, RY, true, STAGES>, 1);      // (a key's shares are added up by one block)
}

// Blocks of 8 rows, or of 32 from 9 rows on.  float32, us with 8 / 32 rows a block, heads of 64: 8 rows of 8 x 4,000 keys 32 / 55, 4 x 2,199..6,454 28 / 33; 12
// rows 55 / 59, 42 / 36; heads of 128: 8 rows 63 / 99, 50 / 59; 12 rows 114 / 103, 72 / 62.
template <typename T>
int dispatch(const KeyWeightArgs& a, cudaStream_t stream) {
  const bool few = a.nh / a.nkv * a.last <= 8;
  if (a.hd <= 128) return few ? run<T, 1, 2>(a, stream) : run<T, 4, 2>(a, stream);
  return few ? run<T, 1, 1>(a, stream) : run<T, 4, 1>(a, stream);
}

}  // namespace

LLG_API int llg_key_weights_tile() { return WEIGHT_TILE; }
LLG_API int llg_key_weights_store_rows() { return STORE_ROWS; }

LLG_API int llg_key_weights_simt(const KeyWeightArgs* args, int dtype, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a)) return 1;
  LLG_REQUIRE(a.hd <= MAX_HD, "key_weights: heads of %d elements (1 to %d)", a.hd, MAX_HD);
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  if (dtype == LLG_F32) return dispatch<float>(a, stream);
  if (dtype == LLG_BF16) return dispatch<__nv_bfloat16>(a, stream);
  return llg_fail("key_weights: unknown dtype %d", dtype);
}
