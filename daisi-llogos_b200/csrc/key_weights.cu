// What the last queries of a step give each cached key (the measure that an eviction goes by), on the CUDA cores: float32 arithmetic, storage
// float32 or bfloat16, head sizes up to 384.
//
// For sequence b of a step and key/value head h, over the rows r = (one of the last min(count, last) queries, head g of the group):
//   p_rj = e^{s_rj - M_r} / L_r over the positions j up to the query's own,  s_rj = scale q_r . k_j
//   weights[slot][h][j] = (j < len_before ? weights[slot][h][j] : 0) + sum_r p_rj
// so a key's entry starts with the step that brings the key, and rows of sequences that are not in the step are left as they were.
//
// A weight needs its row's whole sum, so there are two passes over a (sequence, head)'s keys: the first leaves every block's maximum and sum
// per row, and the block with the last ticket joins them; the second divides.  Few rows (a decode step: the heads of a group) leave their
// scores on the way, 4 bytes a row beside a key's 2 hd bytes, and the second pass reads those; with more rows than STORE_ROWS the
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

// A block: KEYS keys of a (sequence, head), ROWS rows at a time; a thread: 4 rows x KEYS / 16 keys.  SECOND: the rows' ends are known.
template <typename T, bool SECOND>
__global__ void __launch_bounds__(THREADS) key_weights_kernel(KeyWeightArgs a) {
  constexpr int KEYS = SIMT_KEYS, KPT = KEYS / 16;
  extern __shared__ __align__(16) float smem[];
  __shared__ float column[8][KEYS];
  pdl_launch_dependents();
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Rows s = rows_of(a, b, KEYS);
  const int p0 = chunk * KEYS;
  if (p0 >= s.total || s.rows <= 0) return;
  const int kp = (a.hd + 3) / 4 * 4, ks = kp + 4;
  float* Ks = smem;                        // [KEYS][ks]
  float* Qs = Ks + KEYS * ks;              // [ROWS][ks]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T* qg = (const T*)a.q;
  const T* kg = (const T*)a.k_pages;
  const int slot = a.slots[b], most = s.group * a.last;
  const long long pair = (long long)b * a.nkv + h;
  stage<T>(Ks, KEYS, a.hd, kp, ks, [&](int r) -> const T* {
    return p0 + r < s.total ? kg + kv_row(a.page_table, a.table_width, a.table_width, slot, p0 + r, h, a.nkv) * a.hd : nullptr;
  });
  float sum[KPT];
#pragma unroll
  for (int c = 0; c < KPT; ++c) sum[c] = 0.f;
  for (int r0 = 0; r0 < s.rows; r0 += ROWS) {
    __syncthreads();
    stage<T>(Qs, ROWS, a.hd, kp, ks, [&](int r) -> const T* {
      return r0 + r < s.rows ? qg + ((long long)(s.tok0 + (r0 + r) / s.group) * a.nh + h * s.group + (r0 + r) % s.group) * a.hd : nullptr;
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
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = r0 + ty * 4 + r;
      const bool there = row < s.rows;
      const int pos = s.pos0 + row / s.group;                       // the query's own position: it sees the keys up to there
      if (SECOND) {
        if (there) {
          const float2 end = row_end(a, pair * most + row);
#pragma unroll
          for (int c = 0; c < KPT; ++c)
            if (p0 + tx + 16 * c <= pos) sum[c] += share(x[r][c] * a.scale, end);
        }
      } else {
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < KPT; ++c) {
          const int p = p0 + tx + 16 * c;
          x[r][c] = p <= pos ? x[r][c] * a.scale : -INFINITY;
          mx = fmaxf(mx, x[r][c]);
          if (a.scores && there && p < s.total) a.scores[score_at(a, pair * most + row, p, KEYS)] = x[r][c];
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        float l = 0.f;
#pragma unroll
        for (int c = 0; c < KPT; ++c) l += x[r][c] == -INFINITY ? 0.f : expf(x[r][c] - mx);
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
        if (there && tx == 0) leave_stats(a, pair * most + row, chunk, mx, l);
      }
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
      add_weight(a, slot, h, p0 + tid, s.before, t);
    }
  } else {
    join_rows(a, pair, s, (s.total + KEYS - 1) / KEYS);
  }
}

template <typename T>
int run(const KeyWeightArgs& a, cudaStream_t stream) {
  const int ks = (a.hd + 3) / 4 * 4 + 4;
  const size_t smem = sizeof(float) * (size_t)(SIMT_KEYS + ROWS) * ks;
  const dim3 grid(a.chunks, a.nkv, a.n_seqs);
  auto go = [&](void (*kernel)(KeyWeightArgs)) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return llg_fail("key_weights: shared memory %zu: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), smem, stream, a);
    if (e != cudaSuccess) return llg_fail("key_weights: launch: %s", cudaGetErrorString(e));
    return 0;
  };
  if (go(key_weights_kernel<T, false>)) return 1;
  return a.scores ? add_stored(a, SIMT_KEYS, stream) : go(key_weights_kernel<T, true>);
}

}  // namespace

LLG_API int llg_key_weights_keys() { return SIMT_KEYS; }
LLG_API int llg_key_weights_store_rows() { return STORE_ROWS; }

LLG_API int llg_key_weights_simt(const KeyWeightArgs* args, int dtype, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a, SIMT_KEYS)) return 1;
  LLG_REQUIRE(a.hd <= MAX_HD, "key_weights: heads of %d elements (1 to %d)", a.hd, MAX_HD);
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  if (dtype == LLG_F32) return run<float>(a, stream);
  if (dtype == LLG_BF16) return run<__nv_bfloat16>(a, stream);
  return llg_fail("key_weights: unknown dtype %d", dtype);
}
