// Attention of trees of drafted tokens over the paged cache, bfloat16, head sizes in steps of 8 up to 128 for keys and values, on mma.sync
// (m16n8k16, float32 accumulation).  What a node sees is said in cache_args.h, the formula in attention_tree.cu.
//
// The kernel streams the cache: with R query rows (nodes x heads of a group) a key's and a value's 4 hd bytes take 4 R hd flops, so up to 16 rows
// of heads of 128, 32 of heads of 64, the memory system decides the time and mma.sync keeps up beside it (eight sequences of 8,190 keys, heads of
// 128, 16 rows: 59 us, 69 % of the copy bandwidth); more go to attention_tree_tc.cu, heads of other sizes stay.  One tree of 8 nodes behind
// 611 keys, 32 heads of 64 in groups of four: 10 us, the latency of two kernels (11 with the plan behind the wait for the kernel before).  Both on the
// device, twenty calls in a CUDA graph, inputs warm in L2; the short one called by itself takes 13, its host's time.
//
//   copies     A fifth warp brings every key and value tile (one cache page of one key/value head) with TMA boxes of 64 x 64 elements into a
//              ring of stages handed over by mbarriers; head sizes that are no multiple of 64 are filled up with zeros by the boxes.
//   work       All units (sequence, key/value head, row block, key tile) form one list that blocks cut into equal runs (tree_tiles.cuh), so that
//              ragged lengths and trees leave no multiprocessor idle.
//   products   A block's four warps share a tile of 64 keys and 16 WR query rows: WR warps along the rows, 4 / WR along the keys.  A warp's
//              scores stay in registers and become the first operand of the second product.
//   softmax    float32; the running maximum is a whole number of binary orders (as in attention_mma.cu), so rescaling is exact, and the rounding of
//              weights to bfloat16 (the second product's operands are) does not depend on how the list was cut.
//   masks      Only tiles that hold nodes, the tree's end or the window's edge look at bits.  In those a value that is not finite must not meet
//              a weight of zero: a warp that finds one among its keys adds that tile's products up itself, leaving out what a row does not see.
//   joining    A run that ends inside a (sequence, head, row block) leaves partial rows, which a second kernel joins (tree_tiles.cuh).
//
// Every wait on an mbarrier is bounded (llg_attn_tree_mma_status).  No load uses cluster multicast.
#include "tree_tiles.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int WORK_WARPS = 4;
constexpr int THREADS = (WORK_WARPS + 1) * 32;
constexpr int BLOCKS_PER_SM = 2;

__device__ int g_error = 0;   // 0 ok; waits that ran out: 1 tile landed, 2 stage free, 3 copies at the end; 4 shared memory not aligned

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// HDP: the head sizes filled up to 64 or 128.  WR: warps along the rows (1, 2, 4).
template <int HDP, int WR, int STAGES>
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
attn_tree_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, TreeArgs a) {
  constexpr int KB = HDP / 64, TILE_BYTES = KB * TK * 128, KSTEPS = HDP / 16;
  constexpr int WK = WORK_WARPS / WR, KEYS = TK / WK, NT = KEYS / 8;       // warps along the keys, a warp's keys, its score tiles of 8 keys
  constexpr int ROWS = 16 * WR;
  constexpr int SLICE = 16;                                                // columns that the key warps add up at a time
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* Ks = smem;                            // [STAGES][TILE_BYTES]
  unsigned char* Vs = smem + STAGES * TILE_BYTES;
  __shared__ uint64_t full[STAGES], empty[STAGES], work_bar;
  __shared__ Plan plan;
  __shared__ int abort_flag;
  __shared__ int node_depth[LLG_TREE_NODES];
  __shared__ __align__(16) float merge[WK > 1 ? WORK_WARPS : 1][WK > 1 ? 16 : 1][SLICE + 2];
  __shared__ float2 merge_ml[WK > 1 ? WORK_WARPS : 1][16];

  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == WORK_WARPS * 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if ((smem_u32(smem) & 1023u) != 0) {                 // uniform over the block
    if (tid == 0) atomicCAS(&g_error, 0, 4);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], WORK_WARPS);
    }
    mbar_init(&work_bar, WORK_WARPS * 32);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  plan_units<THREADS>(a, ROWS, plan, nullptr, [](int, int, int) { return 0; });
  const int G = a.nh / a.nkv;
  const int units = a.nkv * plan.sums[a.n_seqs];
  const int chunk = (unsigned)(units + gridDim.x - 1) / gridDim.x;
  const int u0 = min(units, (int)blockIdx.x * chunk), u1 = min(units, u0 + chunk);
  const int n_units = u1 - u0;
  // first row of the tile of the run's unit i in the pages, seen as [pages x kv heads x 64]
  auto row_of = [&](int i) -> int {
    if (i >= n_units) return 0;
    const Unit c = locate(plan, a.n_seqs, a.nkv, u0 + i);
    const TreeShape sh = tree_shape(a, plan, c.b);
    return (a.page_table[(long long)sh.slot * a.table_width + (sh.t_first + c.t) % a.ring_pages] * a.nkv + c.kvh) * TK;
  };
  int row = warp == WORK_WARPS ? row_of(lane) : 0;
  pdl_wait();                                          // all before it reads sizes, slots and tables alone, which no kernel of a step writes
  typedef Place<HDP, ROWS> P;
  if (tid == 0) P::notes(a.part, gridDim.x)[blockIdx.x].parts = 0;
  if (u0 >= u1) return;
  volatile int* abortp = &abort_flag;

  if (warp == WORK_WARPS) {
    // ---- copies: the lanes look up the pages of 32 tiles side by side, then each in turn issues its tile's boxes ----
    int issued = 0;
    bool fine = true;
    for (int base = 0; base < n_units && fine; base += 32) {
      if (base > 0) row = row_of(base + lane);
      const int n_here = min(32, n_units - base);
      for (int k = 0; k < n_here && fine; ++k) {
        if (lane == k) {
          const int i = base + k, stage = i % STAGES;
          if (i >= STAGES && !mbar_wait(&empty[stage], ((i / STAGES) - 1) & 1, abortp)) {
            if (!*abortp) { *abortp = 1; atomicCAS(&g_error, 0, 2); }
            fine = false;
          } else {
            mbar_expect_tx(&full[stage], 2 * TILE_BYTES);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              tma_load_2d(smem_u32(Ks + stage * TILE_BYTES + kb * (TK * 128)), &map_k, kb * 64, row, &full[stage]);
              tma_load_2d(smem_u32(Vs + stage * TILE_BYTES + kb * (TK * 128)), &map_v, kb * 64, row, &full[stage]);
            }
          }
        }
        fine = __shfl_sync(0xffffffffu, (int)fine, k) != 0;
        if (fine) ++issued;
      }
    }
    // nothing of this block may be in flight when it ends: the last copies of every stage have landed
    if (lane == 0) {
      for (int i = max(0, issued - STAGES); i < issued; ++i) {
        if (!mbar_wait(&full[i % STAGES], (i / STAGES) & 1, abortp)) {
          const unsigned long long t0 = now_ns();                    // another role gave up: its copies still land
          while (!mbar_try_wait(&full[i % STAGES], (i / STAGES) & 1)) {
            if (now_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_error, 0, 3); break; }
          }
        }
      }
    }
    return;
  }

  // ---- the working warps ------------------------------------------------------------------------------
  const int g = lane >> 2, t4 = lane & 3;
  const int wr = warp / WK, wk = warp - wr * WK;        // rows 16 wr .. + 15, keys KEYS wk .. + KEYS - 1 of a tile
  const float sc = a.scale * LOG2E;
  const bf16* qg = (const bf16*)a.q;
  bf16* out = (bf16*)a.out;
  uint32_t work_phase = 0;
  auto work_sync = [&]() -> bool {                      // the working warps' meeting point: a wait with a limit
    mbar_arrive(&work_bar);
    const bool met = mbar_wait(&work_bar, work_phase & 1, abortp);
    ++work_phase;
    if (!met && !*abortp) { *abortp = 1; atomicCAS(&g_error, 0, 1); }
    return met;
  };
  int i = 0;                                            // tiles consumed so far
  int u = u0;
  while (u < u1) {
    const Unit cur = locate(plan, a.n_seqs, a.nkv, u);
    const TreeShape sh = tree_shape(a, plan, cur.b);
    const int n_seg = min(sh.tiles - cur.t, u1 - u);
    const int row0 = cur.rb * ROWS, n_rows = min(ROWS, sh.n * G - row0);
    // depths of the tree's nodes, for windows (read by tiles with nodes only; the last segment's readers are behind a work_sync)
    if (a.window > 0) {
      for (int k = tid; k < sh.n; k += WORK_WARPS * 32) node_depth[k] = __popcll(a.ancestors[sh.tok0 + k]) - 1;
      if (!work_sync()) return;
    }
    // this thread's rows: 16 wr + g and 8 further
    const bf16* qrow[2];
    long long bits[2];
    int depth[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 16 * wr + g + 8 * e;
      const bool there = r < n_rows;
      const int node = there ? (row0 + r) / G : 0, head = there ? (row0 + r) - node * G : 0;
      qrow[e] = there ? qg + ((long long)(sh.tok0 + node) * a.nh + cur.kvh * G + head) * a.hd : nullptr;
      bits[e] = there ? a.ancestors[sh.tok0 + node] : 0;
      depth[e] = __popcll(bits[e]) - 1;
    }
    uint32_t qf[KSTEPS][4];
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = ks * 16 + 2 * t4 + (e >> 1) * 8;
        qf[ks][e] = qrow[e & 1] && d < a.hd ? *reinterpret_cast<const uint32_t*>(qrow[e & 1] + d) : 0u;
      }
    float o[HDP / 8][4];
#pragma unroll
    for (int j = 0; j < HDP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int j = 0; j < n_seg; ++j, ++i) {
      const int stage = i % STAGES;
      if (!mbar_wait(&full[stage], (i / STAGES) & 1, abortp)) {
        if (!*abortp) { *abortp = 1; atomicCAS(&g_error, 0, 1); }
        return;
      }
      __syncwarp();
      const uint32_t kd = smem_u32(Ks + stage * TILE_BYTES), vd = smem_u32(Vs + stage * TILE_BYTES);
      const int p0 = (sh.t_first + cur.t + j) * TK + wk * KEYS;              // this warp's first key
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
        for (int jp = 0; jp < NT / 2; ++jp) {                                // two tiles of 8 keys per ldmatrix
          uint32_t kb[4];
          const int row = wk * KEYS + jp * 16 + (lane & 7) + (lane >> 4) * 8, ch = 2 * ks + ((lane >> 3) & 1);
          ldmatrix_x4(kb, kd + (ch >> 3) * (TK * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
          mma_16816(s[2 * jp], qf[ks], kb[0], kb[1]);
          mma_16816(s[2 * jp + 1], qf[ks], kb[2], kb[3]);
        }
      const bool mixed = p0 + KEYS > sh.lb || (a.window > 0 && p0 < sh.lb + LLG_TREE_NODES - a.window);      // the same for the warp
      if (mixed) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = e >> 1, at = p0 + n * 8 + 2 * t4 + (e & 1) - sh.lb;
            bool sees;
            if (at < 0) sees = a.window <= 0 || depth[r] - at < a.window;
            else sees = at < sh.n && ((bits[r] >> at) & 1) && (a.window <= 0 || depth[r] - node_depth[at] < a.window);
            s[n][e] = sees ? s[n][e] : -INFINITY;
          }
      }
      float mx[2] = {-INFINITY, -INFINITY}, corr[2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float m_new = fmaxf(m[r], ceilf(mx[r] * sc));
        corr[r] = m_new == -INFINITY ? 1.f : pow2_whole(m[r] - m_new);
        m[r] = m_new;
        l[r] *= corr[r];
      }
      const float ms0 = m[0] == -INFINITY ? 0.f : m[0], ms1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = fast_exp2(fmaf(s[n][e], sc, e >> 1 ? -ms1 : -ms0));
          s[n][e] = p;
          l[e >> 1] += p;
        }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int d = 0; d < HDP / 8; ++d) {
          o[d][0] *= corr[0];
          o[d][1] *= corr[0];
          o[d][2] *= corr[1];
          o[d][3] *= corr[1];
        }
      }
      bool wild = false;
      if (mixed) {
        for (int c = lane; c < KEYS * KB * 8; c += 32) {
          const int row = wk * KEYS + c / (KB * 8), ch = c % (KB * 8);
          const uint4 x = *reinterpret_cast<const uint4*>(Vs + stage * TILE_BYTES + (ch >> 3) * (TK * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
          wild |= not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
        }
        wild = __any_sync(0xffffffffu, wild);
      }
      if (!wild) {
#pragma unroll
        for (int kk = 0; kk < KEYS / 16; ++kk) {
          uint32_t pa[4];
          pa[0] = pack_bf16(s[2 * kk][0], s[2 * kk][1]);
          pa[1] = pack_bf16(s[2 * kk][2], s[2 * kk][3]);
          pa[2] = pack_bf16(s[2 * kk + 1][0], s[2 * kk + 1][1]);
          pa[3] = pack_bf16(s[2 * kk + 1][2], s[2 * kk + 1][3]);
#pragma unroll
          for (int jp = 0; jp < HDP / 16; ++jp) {
            uint32_t vb[4];
            const int row = wk * KEYS + kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, ch = 2 * jp + (lane >> 4);
            ldmatrix_x4_trans(vb, vd + (ch >> 3) * (TK * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
            mma_16816(o[2 * jp], pa, vb[0], vb[1]);
            mma_16816(o[2 * jp + 1], pa, vb[2], vb[3]);
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          for (int k = 0; k < 8; ++k) {                                       // key n * 8 + k: its weights lie in the lanes with t4 = k / 2
            const int row = wk * KEYS + n * 8 + k, from = (lane & ~3) | (k >> 1);
            const float w0 = __shfl_sync(0xffffffffu, k & 1 ? s[n][1] : s[n][0], from);
            const float w1 = __shfl_sync(0xffffffffu, k & 1 ? s[n][3] : s[n][2], from);
#pragma unroll
            for (int d = 0; d < HDP / 8; ++d) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(Vs + stage * TILE_BYTES + (d >> 3) * (TK * 128) + row * 128 + (((d & 7) ^ (row & 7)) << 4) + 4 * t4);
              const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
              if (w0 != 0.f) {
                o[d][0] = fmaf(w0, v.x, o[d][0]);
                o[d][1] = fmaf(w0, v.y, o[d][1]);
              }
              if (w1 != 0.f) {
                o[d][2] = fmaf(w1, v.x, o[d][2]);
                o[d][3] = fmaf(w1, v.y, o[d][3]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
    }

    // ---- the run's result of the rows --------------------------------------------------------------------
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (l[r] != l[r] && m[r] == -INFINITY) m[r] = 0.f;             // scores that are no numbers: the row has to show it
    }
    const int rbs = plan.blocks[cur.b + 1] - plan.blocks[cur.b];
    const unsigned p_first = a.nkv * plan.sums[cur.b] + (cur.kvh * rbs + cur.rb) * sh.tiles;      // the rows' first unit
    const int blk_first = p_first / (unsigned)chunk, blk_last = (p_first + sh.tiles - 1) / (unsigned)chunk;
    const bool whole = blk_first == blk_last;
    const int place = 2 * blockIdx.x + (u > u0);
    if (!whole && cur.t == 0 && tid == 0)
      P::notes(a.part, gridDim.x)[blockIdx.x] = Note{blk_last - blk_first + 1, place, n_rows, row0, sh.tok0, cur.kvh, {0, 0}};
    // two neighbouring columns of a row, already the run's own sum: to the output, or to the run's partial rows
    auto emit = [&](int r, int d, float x, float y, float M, float L) {
      if (r >= n_rows) return;
      if (whole) {
        const float inv = L != 0.f ? 1.f / L : 0.f;
        const int node = (row0 + r) / G, head = (row0 + r) - node * G;
        bf16* dst = out + ((long long)(sh.tok0 + node) * a.nh + cur.kvh * G + head) * a.vd + d;
        if (d < a.vd) *reinterpret_cast<uint32_t*>(dst) = pack_bf16(x * inv, y * inv);      // (value sizes are even)
      } else {
        reinterpret_cast<float2*>(P::sums(a.part, place) + (d >> 2) * ROWS + r)[(d >> 1) & 1] = make_float2(x, y);
        if (d == 0) P::ends(a.part, place)[r] = make_float2(M, L);
      }
    };
    if (WK == 1) {
#pragma unroll
      for (int d = 0; d < HDP / 8; ++d) {
        emit(16 * wr + g, d * 8 + 2 * t4, o[d][0], o[d][1], m[0], l[0]);
        emit(16 * wr + g + 8, d * 8 + 2 * t4, o[d][2], o[d][3], m[1], l[1]);
      }
    } else {
      // the warps along the keys add their results up, a slice of the columns at a time
      if (t4 == 0) {
        merge_ml[warp][g] = make_float2(m[0], l[0]);
        merge_ml[warp][g + 8] = make_float2(m[1], l[1]);
      }
#pragma unroll
      for (int c = 0; c < HDP / SLICE; ++c) {
#pragma unroll
        for (int d = 0; d < SLICE / 8; ++d) {
          *reinterpret_cast<float2*>(&merge[warp][g][d * 8 + 2 * t4]) = make_float2(o[c * (SLICE / 8) + d][0], o[c * (SLICE / 8) + d][1]);
          *reinterpret_cast<float2*>(&merge[warp][g + 8][d * 8 + 2 * t4]) = make_float2(o[c * (SLICE / 8) + d][2], o[c * (SLICE / 8) + d][3]);
        }
        if (!work_sync()) return;
        for (int x = tid; x < ROWS * (SLICE / 2); x += WORK_WARPS * 32) {
          const int r = x / (SLICE / 2), d = (x % (SLICE / 2)) * 2, w0 = (r >> 4) * WK;
          float M = -INFINITY, L = 0.f;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WK; ++w) M = fmaxf(M, merge_ml[w0 + w][r & 15].x);
#pragma unroll
          for (int w = 0; w < WK; ++w) {
            const float2 ml = merge_ml[w0 + w][r & 15];
            if (ml.x == -INFINITY) continue;
            const float f = pow2_whole(ml.x - M);
            const float2 v = *reinterpret_cast<const float2*>(&merge[w0 + w][r & 15][d]);
            L += f * ml.y;
            sum.x += f * v.x;
            sum.y += f * v.y;
          }
          emit(r, c * SLICE + d, sum.x, sum.y, M, L);
        }
        if (!work_sync()) return;
      }
    }
    if (!work_sync()) return;              // node_depth and merge are free again
    u += n_seg;
  }
}

// Blocks of a launch: as many as the GPU holds at once while that leaves a block fewer than about a hundred tiles, more and shorter ones
// beyond (multiprocessors do not stream at the same rate; see attention_decode_tma.cu, which measured this).
int grid_blocks(int n_seqs, int nkv, int row_blocks, int max_len) {
  const long long resident = (long long)BLOCKS_PER_SM * llg_sm_count();
  const long long units = (long long)n_seqs * nkv * row_blocks * ((max_len + TK - 1) / TK);
  long long rounds = units / (resident * 48);
  rounds = rounds < 1 ? 1 : (rounds > 2 ? 2 : rounds);
  const long long most = resident * rounds;
  return (int)(units < most ? (units < 1 ? 1 : units) : most);
}

// Warps along the rows: the fewest that take all rows of a tree, so that short row blocks leave no warp without work.
int row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

template <int HDP, int WR, int STAGES>
int launch(const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t stream) {
  constexpr int smem = 2 * STAGES * (HDP / 64) * TK * 128;
  static unsigned long long allowed = 0;
  cudaError_t e = llg_allow_smem(attn_tree_mma_kernel<HDP, WR, STAGES>, smem, allowed);
  if (e != cudaSuccess) return llg_fail("attn_tree_mma: shared memory %d: %s", smem, cudaGetErrorString(e));
  e = llg_launch(attn_tree_mma_kernel<HDP, WR, STAGES>, dim3(blocks), dim3(THREADS), (size_t)smem, stream, mk, mv, a);
  if (e != cudaSuccess) return llg_fail("attn_tree_mma: launch: %s", cudaGetErrorString(e));
  if (llg_check_launch("attn_tree_mma")) return 1;
  return launch_join<HDP, 16 * WR>(a, blocks, "attn_tree_mma", stream);
}

template <int HDP>
long long scratch_of(int blocks, int wr) {
  return wr == 1 ? Place<HDP, 16>::floats(blocks) : wr == 2 ? Place<HDP, 32>::floats(blocks) : Place<HDP, 64>::floats(blocks);
}

}  // namespace

// 1 when this kernel takes the geometry (bfloat16 only): trees of up to `rows` query rows per key/value head.
LLG_API int llg_attn_tree_mma_supported(int hd, int vd, int n_seqs, int rows, int nkv, int max_len) {
  const int per = 16 * row_warps(rows);
  return hd >= 8 && hd <= 128 && hd % 8 == 0 && vd >= 8 && vd <= 128 && vd % 8 == 0 && n_seqs <= MAX_SEQS &&
         list_fits(n_seqs, nkv, (rows + per - 1) / per, max_len, 1, 0);
}

// Floats of scratch of a launch over trees of up to `rows` query rows per key/value head and sequences of up to `max_len` positions.
LLG_API long long llg_attn_tree_mma_scratch_floats(int n_seqs, int rows, int nkv, int hd, int vd, int max_len) {
  const int wr = row_warps(rows), per = 16 * wr, blocks = grid_blocks(n_seqs, nkv, (rows + per - 1) / per, max_len);
  return hd > 64 || vd > 64 ? scratch_of<128>(blocks, wr) : scratch_of<64>(blocks, wr);
}

LLG_API int llg_attn_tree_mma(const TreeArgs* args, cudaStream_t stream) {
  const TreeArgs& a = *args;
  if (check_tree(a, "attn_tree_mma")) return 1;
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  LLG_REQUIRE(llg_attn_tree_mma_supported(a.hd, a.vd, a.n_seqs, a.max_nodes * (a.nh / a.nkv), a.nkv, a.max_len),
              "attn_tree_mma: heads of %d and %d elements (steps of 8 up to 128), %d sequences of up to %d positions", a.hd, a.vd, a.n_seqs, a.max_len);
  CUtensorMap mk, mv;
  const long long rows = (long long)a.n_pages * a.nkv * TK;
  if (!page_map(a.k_pages, rows, a.hd, &mk) || !page_map(a.v_pages, rows, a.vd, &mv))
    return llg_fail("attn_tree_mma: cuTensorMapEncodeTiled failed or is not available");
  const int all = a.max_nodes * (a.nh / a.nkv), wr = row_warps(all), rbs = (all + 16 * wr - 1) / (16 * wr);
  const int blocks = grid_blocks(a.n_seqs, a.nkv, rbs, a.max_len);
  if (a.hd <= 64 && a.vd <= 64)
    return wr == 1 ? launch<64, 1, 6>(a, mk, mv, blocks, stream) : wr == 2 ? launch<64, 2, 6>(a, mk, mv, blocks, stream)
                                                                         : launch<64, 4, 6>(a, mk, mv, blocks, stream);
  return wr == 1 ? launch<128, 1, 3>(a, mk, mv, blocks, stream) : wr == 2 ? launch<128, 2, 3>(a, mk, mv, blocks, stream)
                                                                        : launch<128, 4, 3>(a, mk, mv, blocks, stream);
}

// Error code recorded when a wait ran out (0 = none); clears it.  Synchronises the device.
LLG_API int llg_attn_tree_mma_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  return v;
}
