// What the last queries of a step give each cached key, bfloat16, head sizes in steps of 8 up to 128, on mma.sync (m16n8k16, float32 accumulation).
// The formula, and why there are two passes, stand in key_weights.cu.
//
// The keys are the rows of the products and the queries their columns: S = K Q^T.  A block takes 128 keys (two pages, brought by TMA boxes of 64
// keys x 64 elements) of a (sequence, key/value head); a warp keeps its 32 keys as operands in registers and goes through the queries 16 at a
// time, so that a query is read from shared memory once a warp and a key once.  A decode step (few rows) streams the keys and is bound by
// that; blocks are short and several to a multiprocessor, so that one's copies run beside another's products.
//
// Waits are bounded (llg_key_weights_mma_status).  No load uses cluster multicast.
#include "tree_tiles.cuh"
#include "key_weights.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int KEYS = 128, PAGES = KEYS / TK, WARPS = 4, THREADS = WARPS * 32;
constexpr int QROWS = 64;                    // query rows in shared memory at a time

__device__ int g_error = 0;                  // 0 ok; 1: a wait for keys ran out; 4: shared memory not aligned

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t swz(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

// HDP: the head size filled up to 64 or 128.  SECOND: the rows' ends are known.
template <int HDP, bool SECOND>
__global__ void __launch_bounds__(THREADS, 4) key_weights_mma_kernel(const __grid_constant__ CUtensorMap map_k, KeyWeightArgs a) {
  constexpr int KB = HDP / 64, KSTEPS = HDP / 16;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* Ks = smem;                              // [PAGES][KB][64 keys][128 bytes]
  unsigned char* Qs = smem + PAGES * KB * TK * 128;      // [KB][rows of a pass][128 bytes]
  __shared__ uint64_t landed;
  __shared__ float2 warp_ml[WARPS][QROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int chunk = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Rows s = rows_of(a, b, KEYS);
  const int p0 = chunk * KEYS;
  if (p0 >= s.total || s.rows <= 0) return;
  if ((smem_u32(smem) & 1023u) != 0) {                   // uniform over the block
    if (tid == 0) atomicCAS(&g_error, 0, 4);
    return;
  }
  const int slot = a.slots[b], most = s.group * a.last;
  if (tid == 0) {
    mbar_init(&landed, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    const int pages = min(PAGES, (s.total - p0 + TK - 1) / TK);
    mbar_expect_tx(&landed, pages * KB * TK * 128);
    for (int g = 0; g < pages; ++g) {
      const int page = a.page_table[(long long)slot * a.table_width + p0 / TK + g];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        tma_load_2d(smem_u32(Ks + (g * KB + kb) * (TK * 128)), &map_k, kb * 64, (page * a.nkv + h) * TK, &landed);
    }
  }
  const long long pair = (long long)b * a.nkv + h;
  const int g = lane >> 2, t4 = lane & 3;
  const float sc = a.scale * LOG2E;
  const bool masked = p0 + KEYS - 1 > s.pos0;            // some query does not see all of the block's keys
  const bf16* qg = (const bf16*)a.q;
  const int pass_rows = min(QROWS, (s.rows + 15) / 16 * 16), q_stride = pass_rows * 128;      // bytes of a 64-wide block of the queries
  uint32_t ka[KSTEPS][2][4];
  float sum[4] = {0.f, 0.f, 0.f, 0.f};                   // keys g, g + 8, g + 16, g + 24 of the warp
  for (int r0 = 0; r0 < s.rows; r0 += QROWS) {
    const int rows = min(QROWS, s.rows - r0), rows16 = (rows + 15) / 16 * 16;
    __syncthreads();                                     // the barrier above is set up; the last rows have been read
    for (int c = tid; c < rows16 * KB * 8; c += THREADS) {
      const int row = c / (KB * 8), ch = c % (KB * 8);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows && ch * 8 < a.hd) {
        const int r = r0 + row, q = r / s.group;
        v = *reinterpret_cast<const uint4*>(qg + ((long long)(s.tok0 + q) * a.nh + h * s.group + r - q * s.group) * a.hd + ch * 8);
      }
      *reinterpret_cast<uint4*>(Qs + (ch >> 3) * q_stride + swz(row, ch & 7)) = v;
    }
    if (r0 == 0) {
      const unsigned long long t0 = now_ns();
      bool ok = true;
      while (ok && !mbar_try_wait(&landed, 0)) ok = now_ns() - t0 < WAIT_LIMIT_NS;
      if (!ok) atomicCAS(&g_error, 0, 1);
      __syncwarp();
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int key = warp * 32 + m * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, ch = 2 * ks + (lane >> 4);
          ldmatrix_x4(ka[ks][m], smem_u32(Ks + ((key >> 6) * KB + (ch >> 3)) * (TK * 128)) + swz(key & 63, ch & 7));
        }
    }
    __syncthreads();
    for (int n0 = 0; n0 < rows16; n0 += 16) {
      float x[2][2][4];                                  // [16 keys][8 queries]: keys g, g + 8, queries 2 t4, 2 t4 + 1
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[m][n][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        uint32_t qb[4];
        const int row = n0 + (lane & 7) + (lane >> 4) * 8, ch = 2 * ks + ((lane >> 3) & 1);
        ldmatrix_x4(qb, smem_u32(Qs + (ch >> 3) * q_stride) + swz(row, ch & 7));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma_16816(x[m][0], ka[ks][m], qb[0], qb[1]);
          mma_16816(x[m][1], ka[ks][m], qb[2], qb[3]);
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int row = r0 + n0 + n * 8 + 2 * t4 + c;
          const bool there = row < s.rows;
          const int pos = masked ? s.pos0 + row / s.group : 0;
          float v[4];                                    // this query's scores of keys g + 8 k
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = x[k >> 1][n][(k & 1) * 2 + c];
            if (masked && p0 + warp * 32 + g + 8 * k > pos) v[k] = -INFINITY;
          }
          if (SECOND) {
            if (there) {
              const float2 end = row_end(a, pair * most + row);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (v[k] != -INFINITY) sum[k] += share(v[k] * a.scale, end);
            }
          } else {
            if (a.scores && there) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int p = p0 + warp * 32 + g + 8 * k;
                if (p < s.total) a.scores[score_at(a, pair * most + row, p, KEYS)] = v[k] * a.scale;
              }
            }
            float mx = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            float l = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) l += v[k] == -INFINITY ? 0.f : fast_exp2((v[k] - mx) * sc);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (g == 0) warp_ml[warp][n0 + n * 8 + 2 * t4 + c] = make_float2(mx * a.scale, l);
          }
        }
    }
    if (!SECOND) {
      __syncthreads();
      for (int r = tid; r < rows; r += THREADS) {
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, warp_ml[w][r].x);
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
          if (warp_ml[w][r].x != -INFINITY) l += warp_ml[w][r].y * fast_exp2((warp_ml[w][r].x - m) * LOG2E);
        leave_stats(a, pair * most + r0 + r, chunk, m, l);
      }
    }
  }
  if (SECOND) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
      sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
      const int p = p0 + warp * 32 + g + 8 * k;
      if (t4 == 0 && p < s.total) add_weight(a, slot, h, p, s.before, sum[k]);
    }
  } else {
    join_rows(a, pair, s, (s.total + KEYS - 1) / KEYS);
  }
}

template <int HDP>
int run(const KeyWeightArgs& a, const CUtensorMap& mk, cudaStream_t stream) {
  const int rows = a.nh / a.nkv * a.last, pass_rows = rows < QROWS ? (rows + 15) / 16 * 16 : QROWS;
  const int smem = (HDP / 64) * (PAGES * TK + pass_rows) * 128;
  const dim3 grid(a.chunks, a.nkv, a.n_seqs);
  auto go = [&](void (*kernel)(CUtensorMap, KeyWeightArgs)) -> int {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return llg_fail("key_weights_mma: shared memory %d: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), (size_t)smem, stream, mk, a);
    if (e != cudaSuccess) return llg_fail("key_weights_mma: launch: %s", cudaGetErrorString(e));
    return llg_check_launch("key_weights_mma");
  };
  if (go(key_weights_mma_kernel<HDP, false>)) return 1;
  return a.scores ? add_stored(a, KEYS, stream) : go(key_weights_mma_kernel<HDP, true>);
}

}  // namespace

LLG_API int llg_key_weights_mma_keys() { return KEYS; }
// 1 when this kernel takes the head size (bfloat16 only).
LLG_API int llg_key_weights_mma_supported(int hd) { return hd >= 8 && hd <= 128 && hd % 8 == 0; }

LLG_API int llg_key_weights_mma(const KeyWeightArgs* args, int n_pages, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a, KEYS)) return 1;
  LLG_REQUIRE(llg_key_weights_mma_supported(a.hd), "key_weights_mma: heads of %d elements (steps of 8 up to 128)", a.hd);
  LLG_REQUIRE((uintptr_t)a.k_pages % 16 == 0 && (uintptr_t)a.q % 16 == 0, "key_weights_mma: storage must be 16-byte aligned");
  LLG_REQUIRE((long long)n_pages * a.nkv * TK < 2147483647LL, "key_weights_mma: too many page rows for a tensor map coordinate");
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  CUtensorMap mk;
  if (!page_map(a.k_pages, (long long)n_pages * a.nkv * TK, a.hd, &mk))
    return llg_fail("key_weights_mma: cuTensorMapEncodeTiled failed or is not available");
  return a.hd <= 64 ? run<64>(a, mk, stream) : run<128>(a, mk, stream);
}

// Error code recorded when a wait ran out (0 = none); clears it.  Synchronises the device.
LLG_API int llg_key_weights_mma_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  return v;
}
