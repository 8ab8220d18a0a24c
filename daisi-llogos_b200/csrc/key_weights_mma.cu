// What the last queries of a step give each cached key, bfloat16, head sizes in steps of 8 up to 128, on mma.sync (m16n8k16, float32 accumulation).
// The formula, and why there are two passes, stand in key_weights.cu.
//
// The queries are the rows of the products, S = Q K^T, and stay in registers: MT tiles of 16 rows a warp, WR warps along the rows and 4 / WR along
// the keys.  A block streams one split's keys of a (sequence, key/value head) through a ring of tiles (a page, by TMA boxes of 64 keys x 64
// elements); several blocks share a multiprocessor, so that one's copies run beside another's products.  A thread keeps the maximum and sum
// of its own keys only, and lanes and warps meet at the split's end: no exchange per tile.  The second pass over many rows adds a key's
// shares up over the rows: in a thread, over the eight lanes that hold the key's other rows by halves (7 exchanges for 8 keys), over
// the warps in shared memory.  (With the keys as rows and every row's maximum and sum exchanged per 32 keys, and the splits joined by the last
// block: a decode step of eight sequences of 8,190 keys 51 us; now 33.)  Heads of 64 and 128 with more than 32 rows go to key_weights_tc.cu.
//
// Waits are bounded (llg_key_weights_mma_status).  No load uses cluster multicast.
#include "tree_tiles.cuh"
#include "key_weights.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;

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

// HDP: the head size filled up to 64 or 128.  MT, WR: above.  SECOND: the rows' ends are known.
template <int HDP, int MT, int WR, int STAGES, bool SECOND>
__global__ void __launch_bounds__(THREADS) key_weights_mma_kernel(const __grid_constant__ CUtensorMap map_k, KeyWeightArgs a) {
  constexpr int KB = HDP / 64, KSTEPS = HDP / 16, TILE_BYTES = KB * TK * 128;
  constexpr int WK = WARPS / WR, KEYS = TK / WK, NT = KEYS / 8, ROWS = 16 * MT * WR;
  extern __shared__ __align__(1024) unsigned char smem[];      // [STAGES][KB][64 keys][128 bytes]
  __shared__ uint64_t full[STAGES];
  __shared__ float2 ends[SECOND ? ROWS : 1], warp_ml[WK][SECOND ? 1 : ROWS];
  __shared__ float column[SECOND ? WR : 1][SECOND ? TK : 1];
  pdl_launch_dependents();
  pdl_wait();
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Rows s = rows_of(a, b);
  const int first = split * a.split_keys, last = min(s.total, first + a.split_keys);
  if (first >= last || s.rows <= 0) return;
  if ((smem_u32(smem) & 1023u) != 0) {                   // uniform over the block
    if (tid == 0) atomicCAS(&g_error, 0, 4);
    return;
  }
  const int slot = a.slots[b], most = s.group * a.last, tiles = (last - first + TK - 1) / TK;
  const int passes = (s.rows + ROWS - 1) / ROWS, n_tiles = passes * tiles;      // each block of rows reads the split's keys again
  const int* table = a.page_table + (long long)slot * a.table_width + first / TK;
  auto request = [&](int i) {                            // one thread
    const int page = table[i % tiles];
    mbar_expect_tx(&full[i % STAGES], TILE_BYTES);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      tma_load_2d(smem_u32(smem + (i % STAGES) * TILE_BYTES + kb * (TK * 128)), &map_k, kb * 64, (page * a.nkv + h) * TK, &full[i % STAGES]);
  };
  if (tid == 0) {
    for (int st = 0; st < STAGES; ++st) mbar_init(&full[st], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < min(STAGES, n_tiles); ++i) request(i);
  }
  __syncthreads();
  const long long pair = (long long)b * a.nkv + h;
  const int g = lane >> 2, t4 = lane & 3, wr = warp / WK, wk = warp - wr * WK;
  const float sc = a.scale * LOG2E;
  const bf16* qg = (const bf16*)a.q;
  int i = 0;                                             // tiles so far
  for (int r0 = 0; r0 < s.rows; r0 += ROWS) {
    // this warp's queries; a thread's rows: 16 tiles of rows apart, g and 8 further
    uint32_t qf[MT][KSTEPS][4];
    int pos[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const bf16* src[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = r0 + (wr * MT + t) * 16 + g + 8 * e, q = row / s.group;
        pos[t][e] = s.pos0 + q;
        src[e] = row < s.rows ? qg + ((long long)(s.tok0 + q) * a.nh + h * s.group + row - q * s.group) * a.hd : nullptr;
      }
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = ks * 16 + 2 * t4 + (e >> 1) * 8;
          qf[t][ks][e] = src[e & 1] && d < a.hd ? *reinterpret_cast<const uint32_t*>(src[e & 1] + d) : 0u;
        }
    }
    float2 end[MT][2];
    float m[MT][2], l[MT][2];                            // of this thread's keys; m in the exponent's unit, a whole number
    if (SECOND) {
      __syncthreads();
      if (tid < ROWS && r0 + tid < s.rows) ends[tid] = row_end(a, pair, s, r0 + tid);
      __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = (wr * MT + t) * 16 + g + 8 * e;
        m[t][e] = -INFINITY;
        l[t][e] = 0.f;
        // a row that is none has a sum that is none: its shares are 0
        end[t][e] = SECOND && r0 + row < s.rows ? ends[row] : make_float2(-INFINITY, 0.f);
        if (SECOND && end[t][e].x == -INFINITY) end[t][e] = make_float2(0.f, 0.f);
      }
    for (int p0 = first; p0 < last; p0 += TK, ++i) {
      const unsigned long long t0 = now_ns();
      bool landed = true;
      while (landed && !mbar_try_wait(&full[i % STAGES], (i / STAGES) & 1)) landed = now_ns() - t0 < WAIT_LIMIT_NS;
      if (!landed) atomicCAS(&g_error, 0, 1);
      __syncwarp();
      const uint32_t kd = smem_u32(smem + (i % STAGES) * TILE_BYTES);
      float x[MT][NT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[t][n][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int jp = 0; jp < NT / 2; ++jp) {
          uint32_t kb[4];
          const int row = wk * KEYS + jp * 16 + (lane & 7) + (lane >> 4) * 8, ch = 2 * ks + ((lane >> 3) & 1);
          ldmatrix_x4(kb, kd + (ch >> 3) * (TK * 128) + swz(row, ch & 7));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma_16816(x[t][2 * jp], qf[t][ks], kb[0], kb[1]);
            mma_16816(x[t][2 * jp + 1], qf[t][ks], kb[2], kb[3]);
          }
        }
      const int w0 = p0 + wk * KEYS;                     // this warp's first key; a thread's: w0 + 8 n + 2 t4 + (e & 1)
      if (w0 + KEYS - 1 > s.pos0) {                      // some query does not see all of them
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (w0 + 8 * n + 2 * t4 + (e & 1) > pos[t][e >> 1]) x[t][n][e] = -INFINITY;
      }
      if (!SECOND) {
        if (a.scores) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = r0 + (wr * MT + t) * 16 + g + 8 * e;
              float* dst = a.scores + score_at(a, pair * most + row, w0 + 2 * t4);      // (a split is whole tiles: there is room behind the last key)
              if (row < s.rows) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(x[t][n][2 * e], x[t][n][2 * e + 1]);
              }
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = x[t][0][2 * e];
#pragma unroll
            for (int n = 0; n < NT; ++n) mx = fmaxf(mx, fmaxf(x[t][n][2 * e], x[t][n][2 * e + 1]));
            const float top = fmaxf(m[t][e], ceilf(mx * sc)), ms = top == -INFINITY ? 0.f : top;
            float sum = l[t][e] * (top == m[t][e] ? 1.f : pow2_whole(m[t][e] - top));
#pragma unroll
            for (int n = 0; n < NT; ++n) sum += fast_exp2(fmaf(x[t][n][2 * e], sc, -ms)) + fast_exp2(fmaf(x[t][n][2 * e + 1], sc, -ms));
            m[t][e] = top;
            l[t][e] = sum;
          }
      } else {
        float sum[2 * NT];                               // of key 8 n + 2 t4 + c at 2 n + c, over this thread's rows
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float y = 0.f;
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float v = x[t][n][2 * e + c];        // -inf: a key behind the query, which a row of no numbers does not reach either
                y += v == -INFINITY ? 0.f : fast_exp2(fmaf(v, sc, -end[t][e].x)) * end[t][e].y;
              }
            sum[2 * n + c] = y;
          }
        // over the eight lanes of a key, by halves: a lane keeps the keys whose place has its bits
#pragma unroll
        for (int o = 0; o < 3; ++o) {
          const int half = (2 * NT) >> (o + 1);
          const bool up = (g >> (2 - o)) & 1;
#pragma unroll
          for (int k = 0; k < half; ++k) {
            const float give = up ? sum[k] : sum[k + half], keep = up ? sum[k + half] : sum[k];
            sum[k] = keep + __shfl_xor_sync(0xffffffffu, give, 16 >> o);
          }
        }
#pragma unroll
        for (int k = 0; k < (2 * NT) / 8; ++k) {
          const int at = g * ((2 * NT) / 8) + k;         // place 2 n + c of what this lane has
          column[SECOND ? wr : 0][SECOND ? wk * KEYS + 8 * (at >> 1) + 2 * t4 + (at & 1) : 0] = sum[k];
        }
      }
      __syncthreads();                                   // the tile has been read by all; the columns are there
      if (tid == 0 && i + STAGES < n_tiles) request(i + STAGES);
      if (SECOND) {
        if (tid < TK && p0 + tid < s.total) {
          float y = 0.f;
#pragma unroll
          for (int w = 0; w < WR; ++w) y += column[SECOND ? w : 0][SECOND ? tid : 0];
          add_weight(a, slot, h, p0 + tid, s.before, y, r0 > 0);
        }
        __syncthreads();
      }
    }
    if (!SECOND) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(m[t][e], __shfl_xor_sync(0xffffffffu, m[t][e], 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          float sum = m[t][e] == -INFINITY ? l[t][e] : l[t][e] * pow2_whole(m[t][e] - top);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (t4 == 0) warp_ml[wk][SECOND ? 0 : (wr * MT + t) * 16 + g + 8 * e] = make_float2(top, sum);
        }
      __syncthreads();
      if (tid < ROWS && r0 + tid < s.rows) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, warp_ml[w][SECOND ? 0 : tid].x);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float2 v = warp_ml[w][SECOND ? 0 : tid];
          sum += v.x == -INFINITY ? v.y : v.y * pow2_whole(v.x - top);
        }
        stats_of(a, pair, split)[r0 + tid] = make_float2(top, sum);
      }
      __syncthreads();
    }
  }
}

template <int HDP, int MT, int WR, int STAGES>
int launch(const KeyWeightArgs& a, const CUtensorMap& mk, cudaStream_t stream) {
  constexpr int smem = STAGES * (HDP / 64) * TK * 128;
  const dim3 grid(a.splits, a.nkv, a.n_seqs);
  static unsigned long long first_allowed = 0, second_allowed = 0;
  auto go = [&](void (*kernel)(CUtensorMap, KeyWeightArgs), unsigned long long& allowed) -> int {
    cudaError_t e = llg_allow_smem(kernel, smem, allowed);
    if (e != cudaSuccess) return llg_fail("key_weights_mma: shared memory %d: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), (size_t)smem, stream, mk, a);
    if (e != cudaSuccess) return llg_fail("key_weights_mma: launch: %s", cudaGetErrorString(e));
    return llg_check_launch("key_weights_mma");
  };
  if (go(key_weights_mma_kernel<HDP, MT, WR, STAGES, false>, first_allowed)) return 1;
  if (a.scores) return add_stored(a, stream);
  if constexpr (WR > 1) return go(key_weights_mma_kernel<HDP, MT, WR, STAGES, true>, second_allowed);
  else return llg_fail("key_weights_mma: a warp's %d keys are fewer than the second pass adds up by halves", TK / WARPS);
}

// Rows of a group's queries: up to 16 and 32 one tile a warp, all warps along the keys or two of them; more: two tiles a warp, four along the rows.
// Without scores on the way up to 16 rows are taken as 17 to 32 are: in the second pass a warp has to have 32 keys.
template <int HDP, int STAGES>
int run(const KeyWeightArgs& a, const CUtensorMap& mk, cudaStream_t stream) {
  const int rows = a.nh / a.nkv * a.last;
  if (rows <= 16 && a.scores) return launch<HDP, 1, 1, STAGES>(a, mk, stream);
  if (rows <= 32) return launch<HDP, 1, 2, STAGES>(a, mk, stream);
  return launch<HDP, 2, 4, STAGES>(a, mk, stream);
}

}  // namespace

// 1 when this kernel takes the head size (bfloat16 only).
LLG_API int llg_key_weights_mma_supported(int hd) { return hd >= 8 && hd <= 128 && hd % 8 == 0; }

LLG_API int llg_key_weights_mma(const KeyWeightArgs* args, int n_pages, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a)) return 1;
  LLG_REQUIRE(!a.scores || (long long)a.nh / a.nkv * a.last <= STORE_ROWS, "key_weights_mma: %d rows of scores are not stored", a.nh / a.nkv * a.last);
  LLG_REQUIRE(llg_key_weights_mma_supported(a.hd), "key_weights_mma: heads of %d elements (steps of 8 up to 128)", a.hd);
  LLG_REQUIRE((uintptr_t)a.k_pages % 16 == 0 && (uintptr_t)a.q % 16 == 0, "key_weights_mma: storage must be 16-byte aligned");
  LLG_REQUIRE((long long)n_pages * a.nkv * TK < 2147483647LL, "key_weights_mma: too many page rows for a tensor map coordinate");
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  CUtensorMap mk;
  if (!page_map(a.k_pages, (long long)n_pages * a.nkv * TK, a.hd, &mk))
    return llg_fail("key_weights_mma: cuTensorMapEncodeTiled failed or is not available");
  return a.hd <= 64 ? run<64, 6>(a, mk, stream) : run<128, 3>(a, mk, stream);
}

// Error code recorded when a wait ran out (0 = none); clears it.  Synchronises the device.
LLG_API int llg_key_weights_mma_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  return v;
}
