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

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int THREADS = 128, ROWS = 32, MAX_HD = 384;

template <typename T>
__device__ __forceinline__ float4 load4(const T* p);
template <>
__device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

template <typename T, typename Row>
__device__ __forceinline__ void stage(float* dst, int rows, int width, int padded, int stride, Row row) {
  if ((width & 3) == 0) {
    const int w4 = padded / 4;
    for (int c = threadIdx.x; c < rows * w4; c += THREADS) {
      const int r = c / w4, d = (c - r * w4) * 4;
      const T* src = row(r);
      *reinterpret_cast<float4*>(dst + r * stride + d) = (src && d < width) ? load4<T>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    for (int c = threadIdx.x; c < rows * padded; c += THREADS) {
      const int r = c / padded, d = c - r * padded;
      const T* src = row(r);
      dst[r * stride + d] = (src && d < width) ? to_f32(src[d]) : 0.f;
    }
  }
}

// A block: a split's keys of a (sequence, head), 64 at a time, ROWS rows at a time; a thread: 4 rows x 4 keys.  SECOND: the rows' ends are known.
template <typename T, bool SECOND>
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
  float* Ks = smem;                        // [KEYS][ks]
  float* Qs = Ks + KEYS * ks;              // [ROWS][ks]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T* qg = (const T*)a.q;
  const T* kg = (const T*)a.k_pages;
  const int slot = a.slots[b], most = s.group * a.last;
  const long long pair = (long long)b * a.nkv + h;
  for (int r0 = 0; r0 < s.rows; r0 += ROWS) {
    __syncthreads();
    stage<T>(Qs, ROWS, a.hd, kp, ks, [&](int r) -> const T* {
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
    for (int p0 = first; p0 < last; p0 += KEYS) {
      __syncthreads();
      stage<T>(Ks, KEYS, a.hd, kp, ks, [&](int r) -> const T* {
        return p0 + r < s.total ? kg + kv_row(a.page_table, a.table_width, a.table_width, slot, p0 + r, h, a.nkv) * a.hd : nullptr;
      });
      __syncthreads();
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
          const float4 k = *reinterpret_cast<const float4*>(Ks + (tx + 16 * c) * ks + d);
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

template <typename T>
int run(const KeyWeightArgs& a, cudaStream_t stream) {
  const int ks = (a.hd + 3) / 4 * 4 + 4;
  const size_t smem = sizeof(float) * (size_t)(WEIGHT_TILE + ROWS) * ks;
  const dim3 grid(a.splits, a.nkv, a.n_seqs);
  auto go = [&](void (*kernel)(KeyWeightArgs)) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return llg_fail("key_weights: shared memory %zu: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), smem, stream, a);
    if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
    return 0;
  };
  if (go(key_weights_kernel<T, false>)) return 1;
  return a.scores ? add_stored(a, stream) : go(key_weights_kernel<T, true>);
}

}  // namespace

LLG_API int llg_key_weights_tile() { return WEIGHT_TILE; }
LLG_API int llg_key_weights_store_rows() { return STORE_ROWS; }

LLG_API int llg_key_weights_simt(const KeyWeightArgs* args, int dtype, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a)) return 1;
  LLG_REQUIRE(a.hd <= MAX_HD, "key_weights: heads of %d elements (1 to %d)", a.hd, MAX_HD);
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  if (dtype == LLG_F32) return run<float>(a, stream);
  if (dtype == LLG_BF16) return run<__nv_bfloat16>(a, stream);
  return llg_fail("key_weights: unknown dtype %d", dtype);
}
