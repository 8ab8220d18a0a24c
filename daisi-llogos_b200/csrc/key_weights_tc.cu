// What the last queries of a step give each cached key, bfloat16, heads of 64 and 128 elements, more than 32 rows, on the 5th-generation tensor cores.
// The formula, and why there are two passes, stand in key_weights.cu.
//
// With 128 rows (32 queries of four heads) a pair of pages is a product of 128 x 128 scores, and what takes the time on mma.sync is the exchange
// between the lanes that hold a row's or a key's scores.  Tensor memory's lanes are the product's rows, so here each pass lays its product
// so that what it adds up lies in one thread: the first S = Q K^T, a thread per query row with the row's maximum and sum; the second S^T = K Q^T, a
// thread per key, which adds up its shares over the rows and writes its entry.  No exchange, and the same two operands in shared
// memory.  A block takes one split of a (sequence, key/value head): a copying warp (TMA boxes of a page, a row block's queries), a warp whose one
// lane issues the products into two buffers of tensor memory, four warps of exponentials.  Two blocks share a multiprocessor (half of tensor
// memory each), so that one's first copies run beside another's exponentials.
//
// What bounds it: a pair of pages is 2,500 to 2,700 cycles of a warp's reads of tensor memory, exponentials and sums, two warps a scheduler, and a
// pass 3 us until its first scores are there, of which the second hides the most: its blocks copy and multiply while the first pass ends.  Four
// prompts of 2,199 to 6,454 tokens, 32 queries, 32 heads of 128 in groups of four: 25 us (on mma.sync 55; the second pass waiting for the
// first with all it does 27, and with splits of 4, 6, 8, 10 and 12 pages then 33, 32, 27, 29, 32).  Scores in registers 64 at a time, where 32
// took 30: 39; a quarter or half of the exponentials as polynomials on the pipe of the products, the same: 30 and 31.
//
// Every wait is bounded (llg_key_weights_tc_status); a role that gives up tells the others, and the warps of exponentials go on without waiting, so that
// all come to the end, where tensor memory is freed.  No load uses cluster multicast.
#include "tree_tiles.cuh"
#include "umma_tiles.cuh"
#include "key_weights.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int LANES = 128;                   // of tensor memory: rows of a row block, keys of a pair of pages
constexpr int LOAD_WARP = LANES / 32, ISSUE_WARP = LOAD_WARP + 1, THREADS = (ISSUE_WARP + 1) * 32;
constexpr int TMEM_COLS = 2 * LANES;         // two buffers of scores
constexpr int CHUNK = 32;                    // scores that a thread has in registers

// 0 ok; waits that ran out: 1 scores, 4 free stage, 5 keys or queries copied, 6 free scores, 7 copies at the end; 3 shared memory not aligned
__device__ int g_error = 0;

__device__ __forceinline__ void chunk_of(uint32_t taddr, float (&x)[CHUNK]) {
  uint32_t part[CHUNK / 16][16];
  warp_whole();
#pragma unroll
  for (int c = 0; c < CHUNK / 16; ++c) tmem_ld16(taddr + 16 * c, part[c]);      // uniform
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < CHUNK; ++k) x[k] = __uint_as_float(part[k / 16][k % 16]);
}

template <int HD, int KST, bool SECOND>
__global__ void __launch_bounds__(THREADS, 2)
key_weights_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, KeyWeightArgs a) {
  constexpr int KB = HD / 64, BLOCK = LANES * 128, Q_BYTES = KB * BLOCK, K_BYTES = KB * BLOCK;      // [KB][128 rows][128 bytes]
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* Qs = smem;
  unsigned char* Ks = smem + Q_BYTES;        // [KST]
  __shared__ uint64_t k_full[KST], k_free[KST], s_full[2], s_free[2], q_full, q_free;
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ __align__(16) float minus_m[SECOND ? LANES : 4], inv_l[SECOND ? LANES : 4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((smem_u32(smem) & 1023u) != 0) {       // uniform over the block
    if (tid == 0) atomicCAS(&g_error, 0, 3);
    return;
  }
  // The first pass's blocks let the second's start when they have waited for all that was launched before and have their tensor memory, so what the
  // second reads of the step's tensors is there without a wait; it waits for the first pass's sums alone.
  if (!SECOND) pdl_wait();
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Rows s = rows_of(a, b);
  const int first = split * a.split_keys, last = min(s.total, first + a.split_keys);
  if (first >= last || s.rows <= 0) return;  // uniform over the block
  if (warp == ISSUE_WARP) {                  // (not ahead of blocks of a kernel before that have yet to take theirs, and then wait for them)
    warp_whole();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == LOAD_WARP * 32) {
    for (int st = 0; st < KST; ++st) {
      mbar_init(&k_full[st], 1);
      mbar_init(&k_free[st], 1);
    }
    for (int e = 0; e < 2; ++e) {
      mbar_init(&s_full[e], 1);
      mbar_init(&s_free[e], LANES / 32);
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_free, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pdl_launch_dependents();                   // (not before: see above)
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base_slot;
  const int slot = a.slots[b], tile_tokens = LANES / s.group, tile_rows = tile_tokens * s.group;
  const int pairs = (last - first + LANES - 1) / LANES, blocks = (s.rows + tile_rows - 1) / tile_rows, n_items = blocks * pairs;
  const long long pair_at = (long long)b * a.nkv + h;
  volatile int* abortp = &abort_flag;
  auto give_up = [&](int code) {
    if (!*abortp) { *abortp = 1; atomicCAS(&g_error, 0, code); }
  };

  if (warp == LOAD_WARP) {
    // ---- copies: the lanes look up the pages of 32 items side by side, then each in turn issues its item's boxes ----
    const int* table = a.page_table + (long long)slot * a.table_width;
    int issued = 0, sent = 0;                // items; row blocks' queries
    bool fine = true;
    for (int i0 = 0; i0 < n_items && fine; i0 += 32) {
      const int i = i0 + lane, rb = i / pairs, p = first + (i - rb * pairs) * LANES;
      int y0 = 0, y1 = -1;
      if (i < n_items) {
        y0 = (table[p / TK] * a.nkv + h) * TK;
        if (p + TK < last) y1 = (table[p / TK + 1] * a.nkv + h) * TK;
      }
      const int n_here = min(32, n_items - i0);
      for (int k = 0; k < n_here && fine; ++k) {
        int queries = 0;
        if (lane == k) {
          const int st = i % KST;
          if (rb * pairs == i) {
            if (rb > 0 && !mbar_wait(&q_free, (rb - 1) & 1, abortp)) {
              give_up(4);
              fine = false;
            } else {
              mbar_expect_tx(&q_full, KB * tile_rows * 128);
#pragma unroll
              for (int kb = 0; kb < KB; ++kb)
                tma_load_3d(smem_u32(Qs + kb * BLOCK), &map_q, kb * 64, h * s.group, s.tok0 + rb * tile_tokens, &q_full);
              queries = 1;
            }
          }
          if (!fine) {
          } else if (i >= KST && !mbar_wait(&k_free[st], (i / KST - 1) & 1, abortp)) {
            give_up(4);
            fine = false;
          } else {
            mbar_expect_tx(&k_full[st], KB * TK * 128 * (y1 < 0 ? 1 : 2));
            const uint32_t to = smem_u32(Ks + st * K_BYTES);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              tma_load_2d(to + kb * BLOCK, &map_k, kb * 64, y0, &k_full[st]);
              if (y1 >= 0) tma_load_2d(to + kb * BLOCK + TK * 128, &map_k, kb * 64, y1, &k_full[st]);
            }
          }
        }
        fine = __shfl_sync(0xffffffffu, (int)fine, k) != 0;
        sent += __shfl_sync(0xffffffffu, queries, k);
        if (fine) ++issued;
      }
    }
    // copies still write into this block's shared memory until their barrier completes
    if (lane == 0) {
      auto drain = [&](uint64_t* bar, uint32_t parity) {
        const unsigned long long t0 = now_ns();
        while (!mbar_try_wait(bar, parity)) {
          if (now_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_error, 0, 7); break; }
        }
      };
      for (int i = max(0, issued - KST); i < issued; ++i) drain(&k_full[i % KST], (i / KST) & 1);
      if (sent > 0) drain(&q_full, (sent - 1) & 1);
    }
  } else if (warp == ISSUE_WARP) {
    // ---- products ------------------------------------------------------------------------------------
    if (elect_one()) {
      constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(LANES >> 3) << 17) | ((uint32_t)(LANES >> 4) << 24);
      bool ok = true;
      auto wait_or_fail = [&](uint64_t* bar, uint32_t parity, int code) {
        if (!ok) return;
        if (!mbar_wait(bar, parity, abortp)) {
          give_up(code);
          ok = false;
        }
      };
      const uint32_t qa = smem_u32(Qs);
      int rb = 0, in = 0;                    // row block, item inside it
      for (int i = 0; i < n_items && ok; ++i) {
        if (in == 0) wait_or_fail(&q_full, rb & 1, 5);
        wait_or_fail(&k_full[i % KST], (i / KST) & 1, 5);
        if (i >= 2) wait_or_fail(&s_free[i & 1], (i / 2 - 1) & 1, 6);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t ka = smem_u32(Ks + (i % KST) * K_BYTES);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t at = (ks >> 2) * BLOCK + (ks & 3) * 32;
          umma_bf16(tmem + (uint32_t)(i & 1) * LANES, desc_kmajor((SECOND ? ka : qa) + at), desc_kmajor((SECOND ? qa : ka) + at), IDESC, ks != 0);
        }
        umma_commit(&s_full[i & 1]);
        umma_commit(&k_free[i % KST]);
        if (++in == pairs) {
          umma_commit(&q_free);
          in = 0;
          ++rb;
        }
      }
    }
  } else {
    // ---- exponentials: thread r owns row r (first pass) or key r of the pair (second) -------------------------
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    const float sc = a.scale * LOG2E;
    int i = 0;
    for (int rb = 0; rb < blocks; ++rb) {
      const int row = rb * tile_rows + tid, n_cols = min(tile_rows, s.rows - rb * tile_rows);
      const bool live = tid < n_cols;
      const int pos = s.pos0 + row / s.group;
      float m = -INFINITY, l = 0.f;
      if (SECOND) {
        if (rb == 0) pdl_wait();
        asm volatile("bar.sync 1, 128;" ::: "memory");      // the row block before has been read
        if (tid < LANES) {
          float2 end = live ? row_end(a, pair_at, s, row) : make_float2(0.f, 0.f);
          if (end.x == -INFINITY) end = make_float2(0.f, 0.f);
          minus_m[SECOND ? tid : 0] = -end.x;
          inv_l[SECOND ? tid : 0] = end.y;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      for (int p0 = first; p0 < last; p0 += LANES, ++i) {
        if (!mbar_wait(&s_full[i & 1], (i >> 1) & 1, abortp)) give_up(1);      // (goes on: the others have to come to the end too)
        warp_whole();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t from = lane_base + (uint32_t)(i & 1) * LANES;
        if (!SECOND) {
          const int sees = live ? min(pos + 1, last) - p0 : 0;      // of the pair's keys
#pragma unroll 1
          for (int c0 = 0; c0 < LANES; c0 += CHUNK) {               // uniform
            if (warp_all(sees <= c0)) break;                        // uniform
            float x[CHUNK];
            chunk_of(from + c0, x);
            if (!warp_all(sees >= c0 + CHUNK)) {
#pragma unroll
              for (int k = 0; k < CHUNK; ++k) x[k] = c0 + k < sees ? x[k] : -INFINITY;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < CHUNK; k += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], x[k + 2 * e], x[k + 2 * e + 1]);
            const float top = fmaxf(m, ceilf(max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * sc)), ms = top == -INFINITY ? 0.f : top;
            const float2 sc2 = make_float2(sc, sc), nms2 = make_float2(-ms, -ms);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int k = 0; k < CHUNK; k += 2) {
              const float2 y = __ffma2_rn(make_float2(x[k], x[k + 1]), sc2, nms2);
              sum[(k >> 1) & 1] = __fadd2_rn(sum[(k >> 1) & 1], make_float2(fast_exp2(y.x), fast_exp2(y.y)));
            }
            l = (top == m ? l : l * pow2_whole(m - top)) + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            m = top;
          }
        } else {
          const int p = p0 + tid, r_first = p > s.pos0 ? (p - s.pos0) * s.group - rb * tile_rows : 0;      // the first of the rows that see this key
          const float2 sc2 = make_float2(sc, sc);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
          for (int c0 = 0; c0 < n_cols; c0 += CHUNK) {              // uniform
            float x[CHUNK];
            chunk_of(from + c0, x);
            float2 w[CHUNK / 2];
#pragma unroll
            for (int k = 0; k < CHUNK; k += 4) {
              const float4 mm = *reinterpret_cast<const float4*>(&minus_m[SECOND ? c0 + k : 0]);
              const float2 y0 = __ffma2_rn(make_float2(x[k], x[k + 1]), sc2, make_float2(mm.x, mm.y));
              const float2 y1 = __ffma2_rn(make_float2(x[k + 2], x[k + 3]), sc2, make_float2(mm.z, mm.w));
              w[k / 2] = make_float2(fast_exp2(y0.x), fast_exp2(y0.y));
              w[k / 2 + 1] = make_float2(fast_exp2(y1.x), fast_exp2(y1.y));
            }
            if (warp_all(r_first <= c0) && c0 + CHUNK <= n_cols) {
#pragma unroll
              for (int k = 0; k < CHUNK; k += 4) {
                const float4 il = *reinterpret_cast<const float4*>(&inv_l[SECOND ? c0 + k : 0]);
                sum[0] = __ffma2_rn(w[k / 2], make_float2(il.x, il.y), sum[0]);
                sum[1] = __ffma2_rn(w[k / 2 + 1], make_float2(il.z, il.w), sum[1]);
              }
            } else {                                                // rows that are none, or do not see the key
#pragma unroll
              for (int k = 0; k < CHUNK; ++k)
                if (c0 + k >= r_first && c0 + k < n_cols) sum[k & 1].x += (k & 1 ? w[k / 2].y : w[k / 2].x) * inv_l[SECOND ? c0 + k : 0];
            }
          }
          l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[i & 1]);
        if (SECOND && p0 + tid < last) add_weight(a, slot, h, p0 + tid, s.before, l, rb > 0);
      }
      if (!SECOND && live) stats_of(a, pair_at, split)[row] = make_float2(m, l);
    }
  }
  // every role comes here, also after a wait that ran out: copies in flight have been waited for above
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == ISSUE_WARP) {
    warp_whole();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
  }
}

template <int HD, int KST>
int launch(const KeyWeightArgs& a, const CUtensorMap& mk, const CUtensorMap& mq, cudaStream_t stream) {
  constexpr int smem = (HD / 64) * (1 + KST) * LANES * 128;
  static_assert(2 * (smem + 4096) <= 227 * 1024 && 3 * smem > 228 * 1024, "two blocks a multiprocessor, which has tensor memory for two");
  const dim3 grid(a.splits, a.nkv, a.n_seqs);
  static unsigned long long first_allowed = 0, second_allowed = 0;
  auto go = [&](void (*kernel)(CUtensorMap, CUtensorMap, KeyWeightArgs), unsigned long long& allowed) -> int {
    cudaError_t e = llg_allow_smem(kernel, smem, allowed);
    if (e != cudaSuccess) return llg_fail("key_weights_tc: shared memory %d: %s", smem, cudaGetErrorString(e));
    e = llg_launch(kernel, grid, dim3(THREADS), (size_t)smem, stream, mk, mq, a);
    if (e != cudaSuccess) return llg_fail("key_weights_tc: launch: %s", cudaGetErrorString(e));
    return llg_check_launch("key_weights_tc");
  };
  if (go(key_weights_tc_kernel<HD, KST, false>, first_allowed)) return 1;
  return go(key_weights_tc_kernel<HD, KST, true>, second_allowed);
}

}  // namespace

// 1 when this kernel takes the geometry (bfloat16 only): more rows than have their scores stored, a group's heads in the lanes of tensor memory.
LLG_API int llg_key_weights_tc_supported(int hd, int group, int last) {
  return (hd == 64 || hd == 128) && group >= 1 && group <= LANES && (long long)group * last > STORE_ROWS;
}

LLG_API int llg_key_weights_tc(const KeyWeightArgs* args, int n_pages, cudaStream_t stream) {
  const KeyWeightArgs& a = *args;
  if (check(a)) return 1;
  LLG_REQUIRE(llg_key_weights_tc_supported(a.hd, a.nh / a.nkv, a.last), "key_weights_tc: heads of %d elements (64 or 128), %d of them a group, %d queries", a.hd,
              a.nh / a.nkv, a.last);
  LLG_REQUIRE((uintptr_t)a.k_pages % 16 == 0 && (uintptr_t)a.q % 16 == 0, "key_weights_tc: storage must be 16-byte aligned");
  LLG_REQUIRE((long long)n_pages * a.nkv * TK < 2147483647LL, "key_weights_tc: too many page rows for a tensor map coordinate");
  const int group = a.nh / a.nkv, tile_rows = LANES / group * group;
  LLG_REQUIRE(((long long)group * a.last + tile_rows - 1) / tile_rows * (a.split_keys / LANES + 1) < 2147483647LL, "key_weights_tc: too many queries");
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  CUtensorMap mk, mq;
  if (!page_map(a.k_pages, (long long)n_pages * a.nkv * TK, a.hd, &mk) || !query_map(a.q, a.n_tokens, a.nh, a.hd, group, LANES / group, &mq))
    return llg_fail("key_weights_tc: cuTensorMapEncodeTiled failed or is not available");
  return a.hd == 64 ? launch<64, 4>(a, mk, mq, stream) : launch<128, 2>(a, mk, mq, stream);
}

// Error code recorded when a wait ran out (0 = none); clears it.  Synchronises the device.
LLG_API int llg_key_weights_tc_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  return v;
}
