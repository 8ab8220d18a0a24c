// Attention of large trees of drafted tokens over the paged cache on the 5th-generation tensor cores (tcgen05), bfloat16, head sizes 64 and 128.
// What a node sees is said in cache_args.h, the formula in attention_tree.cu.
//
// With more than 16 query rows (nodes x heads of a group) of 128 elements, 32 of 64, mma.sync is what takes the time, not the cache.  Here 128 rows are
// the lanes of tensor memory, and a block's two groups of four softmax warps each have scores S[128 x 64] (two buffers) and an accumulator
// O[128 x head] of their own there, a lane that issues their products, and two copying warps for both.  Thread r of a group owns row r, so a row's
// softmax needs no exchange; a group's chain of scores, softmax and product takes about 2,000 cycles a tile, half of them exponentials (attention_tc.cu
// says what of; with two threads a row, which meet once a tile, it took longer).  A tile of queries is as many whole nodes as 128 rows hold, so
// that one TMA box of [nodes][heads of the group] brings it; a row block is one or two of them.  Two (PLAIN): each group takes one, and all key
// tiles: 2,700 to 2,800 cycles a key tile.  One (SPLIT): both groups take it, and every second key tile each: one every 1,660 cycles, where the memory
// system brings one every 1,400.  (Row blocks of 128 alone, all of them SPLIT: every 128 rows read the keys again, sixteen full trees behind up
// to 8,000 keys 277 us.)  Eight trees of 13 to 32 nodes behind 8,190 keys, 32 heads of 128 in groups of four: 59 us, of which 7 lie before the first
// scores; sixteen trees of 64 nodes behind 350 to 7,990 keys, 40 heads in groups of five: 192 us, bound by the groups' chains (61 and 198 with the
// plan and the first page look-ups behind the wait for the kernel before).  Both are the device's share: twenty calls in a CUDA graph, inputs as the call
// before left them in L2; calls one by one, with other work's data in L2, 65 and 209.
//
//   work       The units (sequence, key/value head, row block, key tile) of the batch are one list that blocks, one a multiprocessor, cut into runs
//              of equal weight (PLAIN_WEIGHT, SPLIT_WEIGHT a tile, SEGMENT_WEIGHT a row block); keys, values and queries of a run's next segment are
//              copied while the last one ends.
//   softmax    As in attention_tc.cu: weights 2^(x - M) with a whole number M that is raised only when a tile's weights add up to more than
//              2^14, float32 sums, weights rounded to bfloat16 once, because the second product's operands are: half a step each, which makes results
//              1.4 to 1.5 times as far from 64 bits as weights of 32 bits would (0.0025 of the largest and 0.0017).
//   masks      A tile that holds nodes, the tree's end or the window's edge gives every row a 64-bit word of what it sees.  In such a tile a value
//              that is not finite must not meet a weight of zero: the group looks its values over, and where it finds one adds the tile's products
//              up itself, in tensor memory, leaving out what a row does not see; the issuing lane then leaves that tile out.
//   joining    At a SPLIT segment's end the groups' accumulators are added up; a segment that is not its rows' whole list of keys leaves partial
//              rows, which a second kernel joins (tree_tiles.cuh).
//
// Every wait is bounded (llg_attn_tree_tc_status); every role comes to the block's end, where tensor memory is freed.  No load uses cluster multicast.
#include "tree_tiles.cuh"
#include "umma_tiles.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int BQ = 128;                       // rows of a block: lanes of tensor memory
// what a run's parts take, measured: 2,700 to 2,800 cycles a PLAIN tile, 1,660 a SPLIT tile
constexpr int PLAIN_WEIGHT = 5, SPLIT_WEIGHT = 3, SEGMENT_WEIGHT = 8;
constexpr int GROUPS = 2, WORKERS = GROUPS * BQ;
constexpr int ISSUE_WARP = WORKERS / 32, K_LOAD_WARP = ISSUE_WARP + 1, V_LOAD_WARP = ISSUE_WARP + 2, ISSUE_WARP_2 = ISSUE_WARP + 3;
constexpr int THREADS = (ISSUE_WARP_2 + 1) * 32;
constexpr int TMEM_COLS = 512;
constexpr uint32_t G_COLS = 256, O_COL = 128;       // a group's columns: S 2 x 64, O from column 128

// 0 ok; waits that ran out: 1 scores, 2 accumulator, 4 free stage, 5 tile or queries copied, 6 weights, 7 copies at the end, 8 a meeting; 3 shared memory not aligned
__device__ int g_error = 0;

// A sequence's share of the list: tiles, row blocks of which the first `plain` have more than 128 rows, and the weight of one head.
struct Share {
  int tiles, rbs, plain, weight;
};
// `weigh[b]`: the weight of one head in the sequences before b
__device__ __forceinline__ Share share_of(const Plan& p, const int* weigh, int b) {
  Share s;
  s.rbs = p.blocks[b + 1] - p.blocks[b];
  s.tiles = s.rbs > 0 ? (unsigned)(p.sums[b + 1] - p.sums[b]) / (unsigned)s.rbs : 0;
  s.weight = weigh[b + 1] - weigh[b];
  // weight = tiles (PLAIN_WEIGHT plain + SPLIT_WEIGHT (rbs - plain)) + SEGMENT_WEIGHT rbs
  s.plain = s.tiles > 0 ? ((unsigned)(s.weight - SEGMENT_WEIGHT * s.rbs) / (unsigned)s.tiles - SPLIT_WEIGHT * s.rbs) / (PLAIN_WEIGHT - SPLIT_WEIGHT) : 0;
  return s;
}

// The first unit whose weight begins at w or behind it.
__device__ __forceinline__ int unit_at(const Plan& p, const int* weigh, int n_seqs, int nkv, int w) {
  if (w >= nkv * weigh[n_seqs]) return nkv * p.sums[n_seqs];
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (nkv * weigh[mid] <= w) lo = mid;
    else hi = mid - 1;
  }
  const Share s = share_of(p, weigh, lo);
  const unsigned r = w - nkv * weigh[lo], kvh = r / (unsigned)s.weight, in = r - kvh * s.weight;
  const unsigned block = PLAIN_WEIGHT * s.tiles + SEGMENT_WEIGHT, rb = min(in / block, (unsigned)s.plain), x = in - rb * block;
  const unsigned at = (int)rb < s.plain ? (x + PLAIN_WEIGHT - 1) / PLAIN_WEIGHT : (x + SPLIT_WEIGHT - 1) / SPLIT_WEIGHT;
  // (a row block's last SEGMENT_WEIGHT begins no unit)
  return nkv * p.sums[lo] + kvh * s.tiles * s.rbs + rb * s.tiles + min((unsigned)s.tiles, at);
}

// O = (first ? 0 : O corr) + P V for a tile with values that are not finite: a thread adds up its row from the row's weights in tensor memory, and
// leaves out the keys of no weight.  (A function of its own: its registers are not the main loop's.)
template <int HD>
__device__ __noinline__ void add_by_hand(uint32_t p_at, uint32_t o_at, const unsigned char* values, bool first, float corr) {
  for (int c0 = 0; c0 < HD; c0 += 16) {                                        // uniform
    uint32_t rr[16];
    warp_whole();
    tmem_ld16(o_at + c0, rr);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int x = 0; x < 16; ++x) rr[x] = first ? 0u : __float_as_uint(__uint_as_float(rr[x]) * corr);
    const unsigned char* vb = values + (c0 >> 6) * (TK * 128);
    const int ch = (c0 & 63) >> 3;
    for (int h = 0; h < 2; ++h) {                                              // uniform
      uint32_t pr[16];                                                         // the weights of half of the tile's keys
      warp_whole();
      tmem_ld16(p_at + h * 16, pr);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float w = __uint_as_float(e & 1 ? pr[e >> 1] & 0xffff0000u : pr[e >> 1] << 16);
        if (w == 0.f) continue;
        const int key = h * 32 + e;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint4 y = *reinterpret_cast<const uint4*>(vb + swz(key, ch + q));
          const uint32_t yy[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            rr[q * 8 + 2 * z] = __float_as_uint(fmaf(w, __uint_as_float(yy[z] << 16), __uint_as_float(rr[q * 8 + 2 * z])));
            rr[q * 8 + 2 * z + 1] = __float_as_uint(fmaf(w, __uint_as_float(yy[z] & 0xffff0000u), __uint_as_float(rr[q * 8 + 2 * z + 1])));
          }
        }
      }
    }
    warp_whole();
    tmem_st16(o_at + c0, rr);
  }
}

// QT: tiles of queries that a row block may have (1: SPLIT alone).  KST, VST: stages of keys and of values.
template <int HD, int QT, int KST, int VST>
__global__ void __launch_bounds__(THREADS, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
                    TreeArgs a) {
  static_assert(KST % 2 == 0 && VST % 2 == 0, "where the groups take turns with the tiles, a stage belongs to one of them: a wait for its next phase by parity means "
                "something only to who has seen the last one");
  constexpr int KB = HD / 64, Q_BYTES = KB * BQ * 128, KV_BYTES = KB * TK * 128;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* Qs = smem;
  unsigned char* Ks = Qs + QT * Q_BYTES;             // [KST]
  unsigned char* Vs = Ks + KST * KV_BYTES;           // [VST]
  __shared__ uint64_t k_full[KST], k_free[KST], v_full[VST], v_free[VST];
  __shared__ uint64_t s_full[GROUPS][2], p_ready[GROUPS][2], o_done[GROUPS], q_full, q_free, meet_bar, group_bar[GROUPS];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ int wild[GROUPS][3], leave_out[GROUPS][2];
  __shared__ float2 share[GROUPS][BQ];               // each group's maximum and sum of a row
  __shared__ Plan plan;
  __shared__ int weigh[MAX_SEQS + 1];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((smem_u32(smem) & 1023u) != 0) {               // uniform over the block
    if (tid == 0) atomicCAS(&g_error, 0, 3);
    return;
  }
  if (tid == K_LOAD_WARP * 32) {
    for (int st = 0; st < KST; ++st) {
      mbar_init(&k_full[st], 1);
      mbar_init(&k_free[st], GROUPS);                // (where one group has a tile, its lane arrives for both)
    }
    for (int st = 0; st < VST; ++st) {
      mbar_init(&v_full[st], 1);
      mbar_init(&v_free[st], GROUPS);
    }
    for (int g = 0; g < GROUPS; ++g) {
      mbar_init(&s_full[g][0], 1);
      mbar_init(&s_full[g][1], 1);
      mbar_init(&p_ready[g][0], BQ / 32);
      mbar_init(&p_ready[g][1], BQ / 32);
      mbar_init(&o_done[g], 1);
      mbar_init(&group_bar[g], BQ);
      wild[g][0] = wild[g][1] = wild[g][2] = 0;
      leave_out[g][0] = leave_out[g][1] = 0;
    }
    mbar_init(&q_full, 1);
    mbar_init(&q_free, GROUPS);
    mbar_init(&meet_bar, WORKERS);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int G = a.nh / a.nkv, tile_nodes = BQ / G, tile_rows = tile_nodes * G, block_rows = QT * tile_rows;
  plan_units<THREADS>(a, block_rows, plan, weigh, [&](int rows, int rbs, int tiles) {
    const int split = QT == 1 ? rbs : rbs > 0 && rows - (rbs - 1) * block_rows <= tile_rows;
    return tiles * (PLAIN_WEIGHT * (rbs - split) + SPLIT_WEIGHT * split) + SEGMENT_WEIGHT * rbs;
  });
  // (a run's weight is at least a unit's, so no run between two others is without a unit)
  const int weight = a.nkv * weigh[a.n_seqs];
  const int chunk = max(PLAIN_WEIGHT, (int)((unsigned)(weight + gridDim.x - 1) / gridDim.x));
  const int u0 = unit_at(plan, weigh, a.n_seqs, a.nkv, min(weight, (int)blockIdx.x * chunk));
  const int u1 = unit_at(plan, weigh, a.n_seqs, a.nkv, min(weight, ((int)blockIdx.x + 1) * chunk));
  const int n_units = u1 - u0;                       // (none: every role passes by)
  // What a copying lane needs of the run's unit i: its tile's first row in the pages, seen as [pages x kv heads x 64], and where a segment begins its
  // queries' first token and head, and how many tiles of them (for the values' warp, which brings them).
  struct Copy {
    int row, q_tok, q_head, q_tiles;
  };
  auto copy_of = [&](int i) -> Copy {
    Copy x = {0, 0, 0, 0};
    if (i < n_units) {
      const Unit c = locate(plan, a.n_seqs, a.nkv, u0 + i);
      const TreeShape sh = tree_shape(a, plan, c.b);
      if (warp == V_LOAD_WARP && (i == 0 || c.t == 0)) {
        x.q_tok = sh.tok0 + c.rb * QT * tile_nodes;
        x.q_head = c.kvh * G;
        x.q_tiles = QT > 1 && sh.n - c.rb * QT * tile_nodes > tile_nodes ? 2 : 1;
      }
      const int page = a.page_table[(long long)sh.slot * a.table_width + (sh.t_first + c.t) % a.ring_pages];
      x.row = (page * a.nkv + c.kvh) * TK;
    }
    return x;
  };
  Copy next_copy = {0, 0, 0, 0};
  if (warp == K_LOAD_WARP || warp == V_LOAD_WARP) next_copy = copy_of(lane);
  pdl_wait();                                        // all before it reads sizes, slots and tables alone, which no kernel of a step writes
  if (warp == ISSUE_WARP) {
    warp_whole();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // (not before: a block of the next kernel must not take tensor memory ahead of this one and then wait for it)
  pdl_launch_dependents();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  typedef Place<HD, QT * BQ> P;
  if (tid == 0) P::notes(a.part, gridDim.x)[blockIdx.x].parts = 0;
  const uint32_t tmem = tmem_base_slot;
  volatile int* abortp = &abort_flag;
  auto give_up = [&](int code) {
    if (!*abortp) { *abortp = 1; atomicCAS(&g_error, 0, code); }
  };

  if (warp == K_LOAD_WARP || warp == V_LOAD_WARP) {
    // ---- copies: the lanes look up the pages of 32 tiles side by side, then each in turn issues its tile's boxes ----
    const bool keys = warp == K_LOAD_WARP;
    unsigned char* base = keys ? Ks : Vs;
    uint64_t* full = keys ? k_full : v_full;
    uint64_t* freeb = keys ? k_free : v_free;
    const int stages = keys ? KST : VST;
    const CUtensorMap* map = keys ? &map_k : &map_v;
    if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    // The values' warp brings each segment's queries too, ahead of its first values, when all of the last segment's scores are there.
    int issued = 0, segments = 0;
    bool fine = true;
    for (int first = 0; first < n_units && fine; first += 32) {
      const Copy at = first > 0 ? copy_of(first + lane) : next_copy;
      const int row = at.row, q_tok = at.q_tok, q_head = at.q_head, q_tiles = at.q_tiles;
      const int n_here = min(32, n_units - first);
      for (int k = 0; k < n_here && fine; ++k) {
        int sent = 0;
        if (lane == k) {
          const int i = first + k, st = i % stages;
          if (q_tiles > 0) {
            if (segments > 0 && !mbar_wait(&q_free, (segments - 1) & 1, abortp)) {
              give_up(4);
              fine = false;
            } else {
              mbar_expect_tx(&q_full, q_tiles * KB * tile_rows * 128);
              for (int t = 0; t < q_tiles; ++t)
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                  tma_load_3d(smem_u32(Qs + t * Q_BYTES + kb * (BQ * 128)), &map_q, kb * 64, q_head, q_tok + t * tile_nodes, &q_full);
              sent = 1;
            }
          }
          if (!fine) {
          } else if (i >= stages && !mbar_wait(&freeb[st], (i / stages - 1) & 1, abortp)) {
            give_up(4);
            fine = false;
          } else {
            mbar_expect_tx(&full[st], KV_BYTES);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) tma_load_2d(smem_u32(base + st * KV_BYTES + kb * (TK * 128)), map, kb * 64, row, &full[st]);
          }
        }
        fine = __shfl_sync(0xffffffffu, (int)fine, k) != 0;
        segments += __shfl_sync(0xffffffffu, sent, k);
        if (fine) ++issued;
      }
    }
    // copies still write into this block's shared memory until their barrier completes
    if (lane == 0) {
      for (int i = max(0, issued - stages); i < issued; ++i) {
        const unsigned long long t0 = now_ns();
        while (!mbar_try_wait(&full[i % stages], (i / stages) & 1)) {
          if (now_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_error, 0, 7); break; }
        }
      }
      if (segments > 0) {
        const unsigned long long t0 = now_ns();
        while (!mbar_try_wait(&q_full, (segments - 1) & 1)) {
          if (now_ns() - t0 > WAIT_LIMIT_NS) { atomicCAS(&g_error, 0, 7); break; }
        }
      }
    }
  } else if (warp == ISSUE_WARP || warp == ISSUE_WARP_2) {
    // ---- products: a lane per group issues them -------------------------------------------------------
    if (elect_one()) {
      const int g = warp == ISSUE_WARP ? 0 : 1;
      constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TK >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
      constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
      bool ok = true;
      auto wait_or_fail = [&](uint64_t* bar, uint32_t parity, int code) {
        if (!ok) return;
        if (!mbar_wait(bar, parity, abortp)) {
          give_up(code);
          ok = false;
        }
      };
      // c: the group's tiles so far.  Scores into buffer c % 2, which O += P(c-2) V(c-2) has read by then; a segment's first tile comes
      // when all of the earlier ones are done, and waits for the last of them (a wait by parity sees one phase back).
      auto issue_scores = [&](int i, int c, uint32_t qa, bool first, bool plain) {
        wait_or_fail(&k_full[i % KST], (i / KST) & 1, 5);
        if (first ? c >= 1 : c >= 2) wait_or_fail(&o_done[g], (first ? c - 1 : c) & 1, 6);
        if (!ok) return;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t ka = smem_u32(Ks + (i % KST) * KV_BYTES);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          const uint32_t blk = ks >> 2, kk = ks & 3;
          umma_bf16(tmem + g * G_COLS + (uint32_t)(c & 1) * TK, desc_kmajor(qa + blk * (BQ * 128) + kk * 32),
                    desc_kmajor(ka + blk * (TK * 128) + kk * 32), IDESC_S, ks != 0);
        }
        umma_commit(&s_full[g][c & 1]);
        umma_commit(&k_free[i % KST]);
        if (!plain) umma_commit(&k_free[i % KST]);
      };
      int i0 = 0, c = 0;
      for (int seg = 0; i0 < n_units && ok; ++seg) {
        const Unit cur = locate(plan, a.n_seqs, a.nkv, u0 + i0);
        const Share sh = share_of(plan, weigh, cur.b);
        const int i1 = min(n_units, i0 + sh.tiles - cur.t);
        const bool plain = cur.rb < sh.plain;
        const int step = plain ? 1 : 2;
        const uint32_t qa = smem_u32(Qs + (plain ? g * Q_BYTES : 0));
        int i = i0 + (plain ? 0 : g);
        bool started = false;
        // Both lanes wait for every segment's queries and both give them back, with tiles or without: neither falls behind by a phase, and who
        // has seen the queries knows that the keys of all earlier segments were used.
        wait_or_fail(&q_full, seg & 1, 5);
        if (i < i1) issue_scores(i, c, qa, true, plain);
        if (ok && i + step >= i1) umma_commit(&q_free);
        for (; i < i1 && ok; i += step, ++c) {
          if (i + step < i1) {
            issue_scores(i + step, c + 1, qa, false, plain);
            if (ok && i + 2 * step >= i1) umma_commit(&q_free);
          }
          // (weights first: behind them lie the meetings of earlier segments, so all of their values were used)
          wait_or_fail(&p_ready[g][c & 1], (c >> 1) & 1, 6);
          wait_or_fail(&v_full[i % VST], (i / VST) & 1, 5);
          // (the last tile's product is waited for at the next segment's begin: the one ahead of it has to be done while that can be told)
          if (c >= 1 && i + step >= i1) wait_or_fail(&o_done[g], (c - 1) & 1, 6);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (*reinterpret_cast<volatile int*>(&leave_out[g][c & 1])) {
            umma_commit(&o_done[g]);                   // the group has added this tile up itself, and gives its values back itself
          } else {
            const uint32_t pa = tmem + g * G_COLS + (uint32_t)(c & 1) * TK, va = smem_u32(Vs + (i % VST) * KV_BYTES);
#pragma unroll
            for (int kk = 0; kk < TK / 16; ++kk)
              umma_bf16_ts(tmem + g * G_COLS + O_COL, pa + kk * 8, desc_mnmajor(va + kk * 2048, TK * 128), IDESC_O, started || kk != 0);
            umma_commit(&o_done[g]);
            umma_commit(&v_free[i % VST]);
            if (!plain) umma_commit(&v_free[i % VST]);
          }
          started = true;
        }
        i0 = i1;
      }
    }
  } else {
    // ---- softmax: thread r of group g owns row r -------------------------------------------------------
    const int g = tid / BQ, r = tid % BQ, gw = (tid % BQ) >> 5;       // gw: warp inside the group = its lane quarter
    const uint32_t quarter = (uint32_t)(gw * 32) << 16, lane_base = tmem + g * G_COLS + quarter;
    const float sc = a.scale * LOG2E;
    const float sum_bound = 16384.0f;
    uint32_t meets = 0, group_meets = 0;
    // Meetings of all softmax threads, and of a group's: waits with a limit.  The answer is the warp's.
    auto meet = [&]() -> bool {
      mbar_arrive(&meet_bar);
      const bool met = mbar_wait(&meet_bar, meets & 1, abortp);
      ++meets;
      if (!met) give_up(8);
      return warp_all(met);
    };
    auto group_meet = [&]() -> bool {
      mbar_arrive(&group_bar[g]);
      const bool met = mbar_wait(&group_bar[g], group_meets & 1, abortp);
      ++group_meets;
      if (!met) give_up(8);
      return warp_all(met);
    };
    int looked = 0;                                     // tiles that the group has looked over for values that are not finite
    int i0 = 0, c = 0;                                  // c: the group's tiles so far
    bool ok = true;
    // What a thread knows of a segment; the next one's is asked for before the last one ends.
    struct Segment {
      Unit at;
      TreeShape sh;
      Share list;
      bool plain, live;
      int row0, n_rows, mine, node, depth;
      unsigned long long bits;
    };
    auto segment_at = [&](int i) -> Segment {
      Segment x;
      x.at = locate(plan, a.n_seqs, a.nkv, u0 + i);
      x.list = share_of(plan, weigh, x.at.b);
      x.sh = tree_shape(a, plan, x.at.b);
      x.plain = x.at.rb < x.list.plain;                 // the same for the block
      x.row0 = x.at.rb * block_rows;
      x.n_rows = min(block_rows, x.sh.n * G - x.row0);
      x.mine = x.plain ? g * tile_rows + r : r;         // this thread's row of the row block
      x.live = r < tile_rows && x.mine < x.n_rows;
      x.node = x.live ? (x.row0 + x.mine) / G : 0;
      x.bits = x.live ? (unsigned long long)a.ancestors[x.sh.tok0 + x.node] : 0ull;
      x.depth = __popcll(x.bits) - 1;
      return x;
    };
    Segment next;
    if (n_units > 0) next = segment_at(0);
    while (i0 < n_units && ok) {
      const Unit cur = next.at;
      const TreeShape sh = next.sh;
      const Share list = next.list;
      const bool plain = next.plain, live = next.live;
      const int row0 = next.row0, n_rows = next.n_rows, mine = next.mine, node = next.node, depth = next.depth;
      const int head = cur.kvh * G + row0 + mine - node * G;
      const int i1 = min(n_units, i0 + sh.tiles - cur.t), step = plain ? 1 : 2;
      unsigned long long bits = next.bits;
      bits &= sh.n >= 64 ? ~0ull : (1ull << sh.n) - 1;
      if (a.window > 0 && depth + 1 >= a.window)        // of what it sees, what stands less than a window above it (a node of no bits: at -1)
        for (int j = 0; j < sh.n; ++j)
          if (((bits >> j) & 1) && depth - (__popcll(a.ancestors[sh.tok0 + j]) - 1) >= a.window) bits &= ~(1ull << j);
      float m_run = -INFINITY, l_run = 0.f;
      const int own0 = i0 + (plain ? 0 : g);
      for (int i = own0; i < i1; i += step, ++c) {
        const bool first = i == own0, last = i + step >= i1;
        const bool scored = mbar_wait(&s_full[g][c & 1], (c >> 1) & 1, abortp);
        if (!scored) give_up(1);
        ok = warp_all(scored);
        if (!ok) break;                      // uniform
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int p0 = (sh.t_first + cur.t + i - i0) * TK;
        float sv[TK];
        {
          uint32_t r0_[16], r1_[16], r2_[16], r3_[16];
          const uint32_t sa = lane_base + (uint32_t)(c & 1) * TK;
          tmem_ld16(sa, r0_);
          tmem_ld16(sa + 16, r1_);
          tmem_ld16(sa + 32, r2_);
          tmem_ld16(sa + 48, r3_);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            sv[x] = __uint_as_float(r0_[x]);
            sv[16 + x] = __uint_as_float(r1_[x]);
            sv[32 + x] = __uint_as_float(r2_[x]);
            sv[48 + x] = __uint_as_float(r3_[x]);
          }
        }
        const bool mixed = p0 + TK > sh.lb || (a.window > 0 && p0 < sh.lb + LLG_TREE_NODES - a.window);      // the same for the block
        bool by_hand = false;
        if (mixed) {                          // uniform
          const int shift = sh.lb - p0;      // places of the tile that are cached keys
          unsigned long long cached = shift >= 64 ? ~0ull : shift > 0 ? (1ull << shift) - 1 : 0ull;
          if (a.window > 0) {
            const int from = shift + depth - a.window + 1;
            cached = from >= 64 ? 0ull : from > 0 ? cached & (~0ull << from) : cached;
          }
          const unsigned long long nodes = shift >= 64 ? 0ull : shift >= 0 ? bits << shift : shift > -64 ? bits >> -shift : 0ull;
          const unsigned long long seen = cached | nodes;
          const uint32_t s_lo = (uint32_t)seen, s_hi = (uint32_t)(seen >> 32);
#pragma unroll
          for (int x = 0; x < TK; ++x) sv[x] = ((x < 32 ? s_lo : s_hi) >> (x & 31)) & 1 ? sv[x] : -INFINITY;
          // the group looks the tile's values over
          const bool landed = mbar_wait(&v_full[i % VST], (i / VST) & 1, abortp);
          if (!landed) give_up(5);
          bool found = false;
          if (landed) {
            const uint4* v = reinterpret_cast<const uint4*>(Vs + (i % VST) * KV_BYTES);
#pragma unroll
            for (int x = 0; x < KV_BYTES / 16 / BQ; ++x) {
              const uint4 y = v[x * BQ + r];
              found |= not_finite(y.x) || not_finite(y.y) || not_finite(y.z) || not_finite(y.w);
            }
          }
          if (found) *reinterpret_cast<volatile int*>(&wild[g][looked % 3]) = 1;
          if (r == 0) *reinterpret_cast<volatile int*>(&wild[g][(looked + 1) % 3]) = 0;      // last read before the meeting ahead of this one
          ok = warp_all(landed);
          ok = group_meet() && ok;
          if (!ok) break;                    // uniform
          by_hand = *reinterpret_cast<volatile int*>(&wild[g][looked % 3]) != 0;
          ++looked;
        }
        uint32_t pk[TK / 2];
        float psum;
        auto weights = [&](float m) {
          const float ms = m == -INFINITY ? 0.f : m;
          const float2 sc2 = make_float2(sc, sc), nms2 = make_float2(-ms, -ms);
          float2 ps2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < TK / 2; ++e) {
            const float2 x = __ffma2_rn(make_float2(sv[2 * e], sv[2 * e + 1]), sc2, nms2);
            const float2 w = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            ps2[e & 1] = __fadd2_rn(ps2[e & 1], w);
            pk[e] = pack_bf16(w.x, w.y);
          }
          psum = (ps2[0].x + ps2[0].y) + (ps2[1].x + ps2[1].y);
        };
        float corr = 1.f;
        bool fits = false, rescale = false;              // the latter one answer for the warp
#pragma unroll 1
        for (int pass = first; ; ++pass) {
          if (pass == 1) {
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int x = 0; x < TK; x += 8) {
#pragma unroll
              for (int k = 0; k < 4; ++k) mx4[k] = max3(mx4[k], sv[x + 2 * k], sv[x + 2 * k + 1]);
            }
            const float mxs = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
            const float m_new = fits ? m_run : fmaxf(m_run, ceilf(mxs));
            corr = m_new == m_run || m_new == -INFINITY || !live ? 1.f : pow2_whole(m_run - m_new);
            m_run = m_new;
            rescale = !warp_all(corr == 1.f);
          }
          weights(m_run);
          fits = !live || (m_run != -INFINITY && psum <= sum_bound);      // (a row that is none holds whatever lay in shared memory)
          if (pass == 1 || warp_all(fits)) break;        // uniform
        }
        l_run = l_run * corr + psum;
        warp_whole();
#pragma unroll
        for (int c16 = 0; c16 < TK / 32; ++c16)          // uniform
          tmem_st16(lane_base + (uint32_t)(c & 1) * TK + c16 * 16, reinterpret_cast<const uint32_t(&)[16]>(pk[c16 * 16]));
        // O += P(c-1) V(c-1) has finished: before O is touched, and at the segment's last tile (a wait by parity sees one phase back)
        const bool touch = !first && (rescale || by_hand);
        if (touch || (!first && last)) {
          const bool added = mbar_wait(&o_done[g], (c - 1) & 1, abortp);
          if (!added) give_up(2);
          ok = warp_all(added);
          if (!ok) break;                                // uniform
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (by_hand) {                                   // uniform
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          add_by_hand<HD>(lane_base + (uint32_t)(c & 1) * TK, lane_base + O_COL, Vs + (i % VST) * KV_BYTES, first, corr);
        } else if (touch) {                              // uniform
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 16) {          // uniform
            uint32_t rr[16];
            warp_whole();
            tmem_ld16(lane_base + O_COL + c0, rr);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int x = 0; x < 16; ++x) rr[x] = __float_as_uint(__uint_as_float(rr[x]) * corr);
            tmem_st16(lane_base + O_COL + c0, rr);
          }
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        if (mixed) {                                     // uniform: only such a tile changes what the issuing lane reads here
          if (by_hand) {
            ok = group_meet();                           // all of the group have read the values
            if (!ok) break;                              // uniform
            if (r == 0) {
              mbar_arrive(&v_free[i % VST]);
              if (!plain) mbar_arrive(&v_free[i % VST]);
            }
          }
          if (r == 0) *reinterpret_cast<volatile int*>(&leave_out[g][c & 1]) = by_hand;
        } else if (r == 0) {
          *reinterpret_cast<volatile int*>(&leave_out[g][c & 1]) = 0;
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[g][c & 1]);
        if (last) {
          const bool added = mbar_wait(&o_done[g], c & 1, abortp);
          if (!added) give_up(2);
          ok = warp_all(added);
        }
      }
      if (!ok) break;                                    // uniform
      if (i1 < n_units) next = segment_at(i1);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // ---- the segment's result ---------------------------------------------------------------------------
      if (l_run != l_run && m_run == -INFINITY) m_run = 0.f;       // scores that are no numbers: the row has to show it
      const int each = plain ? PLAIN_WEIGHT : SPLIT_WEIGHT, block = (cur.rb < list.plain || QT > 1 ? PLAIN_WEIGHT : SPLIT_WEIGHT) * list.tiles + SEGMENT_WEIGHT;
      const unsigned w_first = a.nkv * weigh[cur.b] + cur.kvh * list.weight + cur.rb * block;      // (of two kinds only the last is not PLAIN)
      const int blk_first = w_first / (unsigned)chunk, blk_last = (w_first + (list.tiles - 1) * each) / (unsigned)chunk;
      const bool whole = blk_first == blk_last;
      const int place = 2 * blockIdx.x + (i0 > 0);
      if (!whole && cur.t == 0 && tid == 0)
        P::notes(a.part, gridDim.x)[blockIdx.x] = Note{blk_last - blk_first + 1, place, n_rows, row0, sh.tok0, cur.kvh, {0, 0}};
      float M = m_run, L = l_run, w0 = 1.f, w1 = 0.f;
      bool some0 = m_run != -INFINITY, some1 = false;   // (an accumulator without a tile holds anything)
      uint32_t from0 = lane_base + O_COL, from1 = 0;
      if (!plain) {                                     // uniform: the groups meet, and each thread takes half of its row's columns
        share[g][r] = make_float2(m_run, l_run);
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        ok = meet();
        if (!ok) break;                                 // uniform
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const float2 ml0 = share[0][r], ml1 = share[1][r];
        M = fmaxf(ml0.x, ml1.x);
        some0 = ml0.x != -INFINITY;
        some1 = ml1.x != -INFINITY;
        w0 = some0 ? pow2_whole(ml0.x - M) : 0.f;
        w1 = some1 ? pow2_whole(ml1.x - M) : 0.f;
        L = ml0.y * w0 + ml1.y * w1;
        from0 = tmem + O_COL + quarter;
        from1 = from0 + G_COLS;
      }
      const float inv = !whole ? 1.f : L != 0.f ? 1.f / L : 0.f;
      bf16* dst = (bf16*)a.out + ((long long)(sh.tok0 + node) * a.nh + head) * HD;
      if (!whole && live && (plain || g == 0)) P::ends(a.part, place)[mine] = make_float2(M, L);
#pragma unroll 1
      for (int c0 = plain ? 0 : g * (HD / 2); c0 < (plain ? HD : (g + 1) * (HD / 2)); c0 += 16) {       // uniform
        uint32_t r0_[16], r1_[16];
        warp_whole();
        tmem_ld16(from0 + c0, r0_);
        if (!plain) tmem_ld16(from1 + c0, r1_);          // uniform
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        float o[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          o[x] = some0 ? w0 * __uint_as_float(r0_[x]) : 0.f;
          if (!plain && some1) o[x] = fmaf(w1, __uint_as_float(r1_[x]), o[x]);
          o[x] *= inv;
        }
        if (live && whole) {
          uint4 v0, v1;
          v0.x = pack_bf16(o[0], o[1]); v0.y = pack_bf16(o[2], o[3]); v0.z = pack_bf16(o[4], o[5]); v0.w = pack_bf16(o[6], o[7]);
          v1.x = pack_bf16(o[8], o[9]); v1.y = pack_bf16(o[10], o[11]); v1.z = pack_bf16(o[12], o[13]); v1.w = pack_bf16(o[14], o[15]);
          *reinterpret_cast<uint4*>(dst + c0) = v0;
          *reinterpret_cast<uint4*>(dst + c0 + 8) = v1;
        } else if (live) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            P::sums(a.part, place)[(c0 / 4 + q) * (QT * BQ) + mine] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");      // the next segment's products overwrite what was read
      __syncwarp();
      if (!plain) ok = meet();                           // uniform: shares and both accumulators have been read
      i0 = i1;
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

// Tiles of queries that a row block may have: trees of one tile leave its place to another pair of key stages.
int query_tiles(int nodes, int group) { return nodes <= BQ / group ? 1 : 2; }

int grid_blocks(const TreeArgs& a) {
  const int per = query_tiles(a.max_nodes, a.nh / a.nkv) * (BQ / (a.nh / a.nkv));
  const long long units = (long long)a.n_seqs * a.nkv * ((a.max_nodes + per - 1) / per) * ((a.max_len + TK - 1) / TK), most = llg_sm_count();
  return (int)(units < most ? (units < 1 ? 1 : units) : most);
}

template <int HD, int QT, int KST, int VST>
int launch(const TreeArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, cudaStream_t stream) {
  constexpr int smem = (HD / 64) * (QT * BQ * 128 + (KST + VST) * TK * 128);
  static_assert(smem > 116 * 1024, "more than half a multiprocessor's: tensor memory is a block's alone");
  const int blocks = grid_blocks(a);
  static unsigned long long allowed = 0;
  cudaError_t e = llg_allow_smem(attn_tree_tc_kernel<HD, QT, KST, VST>, smem, allowed);
  if (e != cudaSuccess) return llg_fail("attn_tree_tc: shared memory %d: %s", smem, cudaGetErrorString(e));
  e = llg_launch(attn_tree_tc_kernel<HD, QT, KST, VST>, dim3(blocks), dim3(THREADS), (size_t)smem, stream, mk, mv, mq, a);
  if (e != cudaSuccess) return llg_fail("attn_tree_tc: launch: %s", cudaGetErrorString(e));
  if (llg_check_launch("attn_tree_tc")) return 1;
  return launch_join<HD, QT * BQ>(a, blocks, "attn_tree_tc", stream);
}

}  // namespace

// 1 when this kernel takes the geometry (bfloat16 only): trees of up to `nodes` nodes.
LLG_API int llg_attn_tree_tc_supported(int hd, int vd, int n_seqs, int group, int nodes, int nkv, int max_len) {
  if (!((hd == 64 || hd == 128) && vd == hd && n_seqs <= MAX_SEQS && group >= 1 && group <= BQ)) return 0;
  const int per = query_tiles(nodes, group) * (BQ / group);
  return list_fits(n_seqs, nkv, (nodes + per - 1) / per, max_len, PLAIN_WEIGHT, SEGMENT_WEIGHT);
}

// Floats of scratch of a launch over trees of up to `nodes` nodes and sequences of up to `max_len` positions.
LLG_API long long llg_attn_tree_tc_scratch_floats(int n_seqs, int nodes, int nkv, int group, int hd, int max_len) {
  TreeArgs a = {};
  a.n_seqs = n_seqs;
  a.max_nodes = nodes;
  a.nkv = nkv;
  a.nh = nkv * group;
  a.max_len = max_len;
  const int blocks = grid_blocks(a);
  if (query_tiles(nodes, group) == 1) return hd == 64 ? Place<64, BQ>::floats(blocks) : Place<128, BQ>::floats(blocks);
  return hd == 64 ? Place<64, 2 * BQ>::floats(blocks) : Place<128, 2 * BQ>::floats(blocks);
}

LLG_API int llg_attn_tree_tc(const TreeArgs* args, cudaStream_t stream) {
  const TreeArgs& a = *args;
  if (check_tree(a, "attn_tree_tc")) return 1;
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  LLG_REQUIRE(llg_attn_tree_tc_supported(a.hd, a.vd, a.n_seqs, a.nh / a.nkv, a.max_nodes, a.nkv, a.max_len),
              "attn_tree_tc: heads of %d and %d elements (64 or 128, the same), %d of them a group (at most %d), %d sequences of up to %d positions", a.hd, a.vd,
              a.nh / a.nkv, BQ, a.n_seqs, a.max_len);
  CUtensorMap mk, mv, mq;
  const long long rows = (long long)a.n_pages * a.nkv * TK;
  if (!page_map(a.k_pages, rows, a.hd, &mk) || !page_map(a.v_pages, rows, a.vd, &mv) || !query_map(a.q, a.n_tokens, a.nh, a.hd, a.nh / a.nkv, BQ / (a.nh / a.nkv), &mq))
    return llg_fail("attn_tree_tc: cuTensorMapEncodeTiled failed or is not available");
  if (query_tiles(a.max_nodes, a.nh / a.nkv) == 1)
    return a.hd == 64 ? launch<64, 1, 8, 8>(a, mk, mv, mq, stream) : launch<128, 1, 6, 4>(a, mk, mv, mq, stream);
  return a.hd == 64 ? launch<64, 2, 8, 8>(a, mk, mv, mq, stream) : launch<128, 2, 4, 4>(a, mk, mv, mq, stream);
}

// Error code recorded when a wait ran out (0 = none); clears it.  Synchronises the device.
LLG_API int llg_attn_tree_tc_status() {
  int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_error, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
  return v;
}
