// Attention of trees of drafted tokens over the paged cache on the CUDA cores: float32 arithmetic, storage float32 or bfloat16, any head
// sizes up to 384 for keys and values.  The true 32-bit path, and the fallback for what attention_tree_mma.cu does not take.
//
// Per sequence b, key/value head and query row r = (node i, head g of the group), with s_j = scale q_r . k_j over the visible keys j
// (cache_args.h says which): out_r = sum_j e^{s_j - m} v_j / sum_j e^{s_j - m}; a row that sees nothing gets zeros.  One pass over the keys
// with a running maximum m and sum; a key's weight is exactly nothing where the row does not see it, whatever the key or value holds there
// (positions behind the tree are never read, a node's value that another node does not see is not multiplied by zero).
//
// A block takes ROWS query rows of a (sequence, key/value head) and one of up to n_splits runs of its 32-key tiles, runs of one length for all
// sequences; all heads of a group and all nodes share a tile's keys and values through shared memory, where the next tile's arrive (cp.async)
// while this one's are used.  Products are 4 rows x 2 keys (scores) and 4 rows x 4 elements x 4 keys (values) a thread at a time, two of them an
// instruction, so that a float read from shared memory is used two to eight times; the keys' rows are padded by 16 bytes, which spreads the
// sixteen rows that a half warp reads over all banks.  Runs that share a row block leave partial results (sums, maximum, sum of weights); the
// block that takes the last ticket joins them in their order, four columns of a row a thread and sixteen runs asked for at once, so results do
// not depend on who comes last.  The running maxima are raised, with the exchange that this takes, only when a weight would be more than 2^12 (with
// an exchange per tile the softmax took 2,800 cycles of a tile's 9,300, now 600 of 7,500).  What bounds it: reads of shared memory for the
// products, 2,500 cycles each, with two to three blocks a multiprocessor; 12 us lie before the first tile and in the join.  Three trees of 8 to 12
// nodes behind 735 to 1,878 keys, 32 heads of 64 in groups of four: 37 us (with all of it behind the wait for the kernel before 38, then with 13 splits
// of five tiles 43, 21 of three 37, 32 of two 40.  One product
// an instruction and an exchange per tile, 13 splits: 54.  Without the copies ahead, a division and a page look-up per 16 bytes, and a warp that
// joined a row run by run: 149).
#include "common.cuh"
#include "cache_args.h"
#include "simt_tiles.cuh"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

constexpr int TK = 32;            // keys per tile (half a page)
constexpr int THREADS = 128;
constexpr int MAX_HD = 384;
constexpr int PART_EXTRA = 4;     // a partial row is [vd, filled up to 4] sums, the maximum, the sum of weights, and 2 unused

// RY: rows per thread; a block's 8 rows of threads take 8 RY query rows.  VD: sums per row and thread, in steps of 64 value elements.
// STAGES: tiles in shared memory, 2 where they fit.
template <typename T, int RY, int VD, int STAGES>
__global__ void __launch_bounds__(THREADS) attn_tree_kernel(TreeArgs a) {
  constexpr int ROWS = 8 * RY;
  extern __shared__ __align__(16) float smem[];
  __shared__ long long bits[ROWS];
  __shared__ int depth[ROWS], node_depth[LLG_TREE_NODES];
  __shared__ int is_last;
  pdl_launch_dependents();
  const int kp = (a.hd + 3) / 4 * 4, vp = (a.vd + 3) / 4 * 4;       // padded row sizes
  const int ks = kp + 4, vs = vp + 4;
  float* Qs = smem;                       // [ROWS][ks]
  float* Ks = Qs + ROWS * ks;             // [STAGES][TK][ks]
  float* Vs = Ks + STAGES * TK * ks;      // [STAGES][TK][vs]
  float* Ps = Vs + STAGES * TK * vs;      // [ROWS][TK + 4]
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int G = a.nh / a.nkv;
  const int b = blockIdx.z, split = blockIdx.x;
  const int row_blocks = gridDim.y / a.nkv;
  const int kvh = blockIdx.y / row_blocks, rb = blockIdx.y - kvh * row_blocks;
  const int tok0 = a.cu_tokens[b];
  const int n = min(min(a.cu_tokens[b + 1], a.n_tokens) - tok0, a.max_nodes);
  const int row0 = rb * ROWS, n_rows = min(ROWS, n * G - row0);
  const int lb = a.len_before[b], slot = a.slots[b], total = lb + n;
  const T* qg = (const T*)a.q;
  const T* kg = (const T*)a.k_pages;
  const T* vg = (const T*)a.v_pages;

  const int lo = a.window > 0 ? max(0, lb - a.window) : 0;          // no row sees less than this (a row without any bit has depth -1)
  const int t0 = lo / TK, t_end = (total + TK - 1) / TK;
  // runs of equal length for all sequences, so that short ones have fewer (the second size: of a sequence that is longer than it may be)
  const int per = max(((a.max_len + TK - 1) / TK + a.n_splits - 1) / a.n_splits, (t_end - t0 + a.n_splits - 1) / a.n_splits);
  const int runs = (t_end - t0 + per - 1) / per;
  // (no rows: the same for all blocks of a row block, so nobody waits for a ticket of theirs)
  const bool none = n_rows <= 0 || split >= runs;
  const int t_from = t0 + split * per, t_to = min(t_end, t_from + per);

  // the page of the tile that is asked for next is looked up a tile ahead
  const int* table = a.page_table + (long long)slot * a.table_width;
  auto page_of = [&](int t) { return t < t_to ? table[t / 2 % a.ring_pages] : 0; };
  int page = none ? 0 : page_of(t_from);
  pdl_wait();                             // all before it reads sizes, slots and tables alone, which no kernel of a step writes
  if (none) return;
  for (int i = tid; i < n; i += THREADS) node_depth[i] = __popcll(a.ancestors[tok0 + i]) - 1;
  for (int r = tid; r < ROWS; r += THREADS) {
    const long long mine = r < n_rows ? a.ancestors[tok0 + (row0 + r) / G] : 0;
    bits[r] = mine;
    depth[r] = __popcll(mine) - 1;
  }
  copy_rows<THREADS, T>(Qs, ks, ROWS, a.hd, kp, [&](int r) {
    return r < n_rows ? qg + ((long long)(tok0 + (row0 + r) / G) * a.nh + kvh * G + (row0 + r) % G) * a.hd : nullptr;
  });

  const float sc = a.scale * 1.4426950408889634f;      // maxima and exponents are in binary orders
  float m[RY], l[RY];
  float2 o[RY][VD * 2];
#pragma unroll
  for (int r = 0; r < RY; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < VD * 2; ++e) o[r][e] = make_float2(0.f, 0.f);
  }
  const TileCopy<THREADS> copy_k(kp), copy_v(vp);
  auto request = [&](int t) {              // tile t into its stage: its keys lie in one page, one behind the other
    if (t < t_to) {
      const int p0 = t * TK, st = (t - t_from) % STAGES;
      const long long row = ((long long)page * a.nkv + kvh) * (2 * TK) + p0 % (2 * TK);
      page = page_of(t + 1);
      copy_k(Ks + st * TK * ks, ks, kg + row * a.hd, TK, total - p0, a.hd);
      copy_v(Vs + st * TK * vs, vs, vg + row * a.vd, TK, total - p0, a.vd);
    }
    tile_commit();
  };
  if (STAGES == 2) request(t_from);
  for (int t = t_from; t < t_to; ++t) {
    const int p0 = t * TK;
    __syncthreads();                       // the stage that is filled now has been read
    request(STAGES == 2 ? t + 1 : t);
    tile_wait<STAGES - 1>();
    __syncthreads();
    const float* Kt = Ks + (t - t_from) % STAGES * TK * ks;
    const float* Vt = Vs + (t - t_from) % STAGES * TK * vs;
    float2 s2[RY][2];                      // elements 0, 2, ... and 1, 3, ...
#pragma unroll
    for (int r = 0; r < RY; ++r) s2[r][0] = s2[r][1] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < kp; d += 4) {
      const float4 k0 = *reinterpret_cast<const float4*>(Kt + tx * ks + d);
      const float4 k1 = *reinterpret_cast<const float4*>(Kt + (tx + 16) * ks + d);
#pragma unroll
      for (int r = 0; r < RY; ++r) {
        const float4 q = *reinterpret_cast<const float4*>(Qs + (ty * RY + r) * ks + d);
        s2[r][0] = __ffma2_rn(make_float2(q.x, q.y), make_float2(k0.x, k0.y), s2[r][0]);
        s2[r][1] = __ffma2_rn(make_float2(q.x, q.y), make_float2(k1.x, k1.y), s2[r][1]);
        s2[r][0] = __ffma2_rn(make_float2(q.z, q.w), make_float2(k0.z, k0.w), s2[r][0]);
        s2[r][1] = __ffma2_rn(make_float2(q.z, q.w), make_float2(k1.z, k1.w), s2[r][1]);
      }
    }
    float s[RY][2];
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      s[r][0] = s2[r][0].x + s2[r][0].y;
      s[r][1] = s2[r][1].x + s2[r][1].y;
    }
    // positions that some row may not see: the tree's, those behind it, the window's edge (a word has up to 64 bits, whatever the tree's nodes)
    const bool mixed = p0 + TK > lb || (a.window > 0 && p0 < lb + LLG_TREE_NODES - a.window);
    if (mixed) {
#pragma unroll
      for (int r = 0; r < RY; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = ty * RY + r, j = p0 + tx + 16 * e - lb;
          const bool sees = j < 0 ? a.window <= 0 || depth[row] - j < a.window
                                  : j < n && ((bits[row] >> j) & 1) && (a.window <= 0 || depth[row] - node_depth[j] < a.window);
          s[r][e] = sees ? s[r][e] : -INFINITY;
        }
    }
    // the maxima are raised, by all lanes of a row, only when a weight would be more than 2^12
    bool raise = false;
#pragma unroll
    for (int r = 0; r < RY; ++r) raise |= fmaxf(s[r][0], s[r][1]) * sc > m[r] + 12.f;
    if (__any_sync(0xffffffffu, raise)) {
      float mx[RY];
#pragma unroll
      for (int r = 0; r < RY; ++r) mx[r] = fmaxf(s[r][0], s[r][1]) * sc;
#pragma unroll
      for (int k = 8; k > 0; k >>= 1)
#pragma unroll
        for (int r = 0; r < RY; ++r) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], k));
#pragma unroll
      for (int r = 0; r < RY; ++r) {
        const float m_new = fmaxf(m[r], mx[r]), corr = m_new == -INFINITY ? 1.f : exp2f(m[r] - m_new);
        m[r] = m_new;
        l[r] *= corr;
#pragma unroll
        for (int e = 0; e < VD * 2; ++e) o[r][e] = __fmul2_rn(o[r][e], make_float2(corr, corr));
      }
    }
#pragma unroll
    for (int r = 0; r < RY; ++r) {
      const float ms = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[r][e] = exp2f(fmaf(s[r][e], sc, -ms));       // (of -inf exactly nothing)
        l[r] += s[r][e];
      }
    }
#pragma unroll
    for (int r = 0; r < RY; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) Ps[(ty * RY + r) * (TK + 4) + tx + 16 * e] = s[r][e];
    __syncwarp();                          // a row's weights come from and go to the lanes of one warp
#pragma unroll 2
    for (int j = 0; j < TK; j += 4) {
      float p[RY][4];
#pragma unroll
      for (int r = 0; r < RY; ++r) *reinterpret_cast<float4*>(p[r]) = *reinterpret_cast<const float4*>(Ps + (ty * RY + r) * (TK + 4) + j);
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        const int d = c * 64 + tx * 4;
        if (d < vp) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(Vt + (j + k) * vs + d);
#pragma unroll
            for (int r = 0; r < RY; ++r) {
              if (!mixed || p[r][k] != 0.f) {
                const float2 w = make_float2(p[r][k], p[r][k]);
                o[r][c * 2] = __ffma2_rn(w, make_float2(v.x, v.y), o[r][c * 2]);
                o[r][c * 2 + 1] = __ffma2_rn(w, make_float2(v.z, v.w), o[r][c * 2 + 1]);
              }
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RY; ++r) {
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], k);
    if (l[r] != l[r] && m[r] == -INFINITY) m[r] = 0.f;               // scores that are no numbers: the row has to show it
  }
  T* out = (T*)a.out;
  const int slots_per_row = a.n_splits;
  const long long first_row = ((long long)b * a.nkv + kvh) * a.max_nodes * G + row0;
  const int pw = vp + PART_EXTRA;
#pragma unroll
  for (int r = 0; r < RY; ++r) {
    const int row = ty * RY + r;
    if (row >= n_rows) continue;
    if (runs == 1) {
      T* dst = out + ((long long)(tok0 + (row0 + row) / G) * a.nh + kvh * G + (row0 + row) % G) * a.vd;
      const float inv = l[r] != 0.f ? 1.f / l[r] : 0.f;
#pragma unroll
      for (int e = 0; e < VD * 4; ++e) {
        const int d = (e >> 2) * 64 + tx * 4 + (e & 3);
        if (d < a.vd) dst[d] = from_f32<T>((e & 1 ? o[r][e >> 1].y : o[r][e >> 1].x) * inv);
      }
    } else {
      float* dst = a.part + ((first_row + row) * slots_per_row + split) * pw;
      if (tx == 0) {
        dst[vp] = m[r];
        dst[vp + 1] = l[r];
      }
      if (m[r] == -INFINITY) continue;                              // nothing seen: nobody reads the sums
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        const int d = c * 64 + tx * 4;
        if (d < vp) *reinterpret_cast<float4*>(dst + d) = make_float4(o[r][2 * c].x, o[r][2 * c].y, o[r][2 * c + 1].x, o[r][2 * c + 1].y);
      }
    }
  }
  if (runs == 1) return;
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int* counter = a.counters + (b * a.nkv + kvh) * row_blocks + rb;
    const int ticket = atomicAdd(counter, 1);
    is_last = ticket == runs - 1;
    if (is_last) *counter = 0;
  }
  __syncthreads();
  if (!is_last) return;
  __threadfence();
  const int v4 = vp / 4;
  constexpr int DEEP = 16;                 // runs asked for at once
  for (int x = tid; x < n_rows * v4; x += THREADS) {
    const int row = x / v4, d = (x - row * v4) * 4;
    const float* src = a.part + (first_row + row) * slots_per_row * pw;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < runs; s0 += DEEP) {
      float2 ml[DEEP];
      float4 v[DEEP];
#pragma unroll
      for (int k = 0; k < DEEP; ++k) {
        const float* p = src + (long long)(s0 + k < runs ? s0 + k : 0) * pw;
        ml[k] = s0 + k < runs ? __ldcg(reinterpret_cast<const float2*>(p + vp)) : make_float2(-INFINITY, 0.f);
        v[k] = __ldcg(reinterpret_cast<const float4*>(p + d));
      }
      float top = M;
#pragma unroll
      for (int k = 0; k < DEEP; ++k) top = fmaxf(top, ml[k].x);
      const float f = M == -INFINITY ? 0.f : exp2f(M - top);
      M = top;
      L *= f;
      acc.x *= f;
      acc.y *= f;
      acc.z *= f;
      acc.w *= f;
#pragma unroll
      for (int k = 0; k < DEEP; ++k) {
        if (ml[k].x == -INFINITY) continue;                          // a run in which the row sees nothing has left no sums
        const float w = exp2f(ml[k].x - M);
        L += w * ml[k].y;
        acc.x += w * v[k].x;
        acc.y += w * v[k].y;
        acc.z += w * v[k].z;
        acc.w += w * v[k].w;
      }
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    T* dst = out + ((long long)(tok0 + (row0 + row) / G) * a.nh + kvh * G + (row0 + row) % G) * a.vd + d;
    const float four[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < a.vd) dst[e] = from_f32<T>(four[e]);
  }
}

// Blocks of 8 rows, or of 32 from 9 rows on.  float32, us with 8 / 32 rows a block, heads of 64: 8 rows behind 8 x 4,000 keys 65 / 98, 3 x 735..1,878 19 / 26,
// 1 x 611 12 / 16; 12 rows 120 / 101, 21 / 29, 14 / 17; heads of 128: 8 rows 142 / 233, 27 / 53, 19 / 27; 12 rows 267 / 236, 51 / 56, 20 / 29.
int rows_per_block(int rows) { return rows <= 8 ? 8 : 32; }

template <typename T, int RY, int VD, int STAGES>
int launch(const TreeArgs& a, cudaStream_t stream) {
  const int kp = (a.hd + 3) / 4 * 4 + 4, vp = (a.vd + 3) / 4 * 4 + 4;
  const size_t smem = sizeof(float) * ((size_t)(8 * RY + STAGES * TK) * kp + (size_t)STAGES * TK * vp + 8 * RY * (TK + 4));
  auto kernel = attn_tree_kernel<T, RY, VD, STAGES>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return llg_fail("attn_tree: shared memory %zu: %s", smem, cudaGetErrorString(e));
  const int G = a.nh / a.nkv, blocks = (a.max_nodes * G + 8 * RY - 1) / (8 * RY);
  LLG_REQUIRE((long long)blocks * a.nkv <= 65535 && a.n_seqs <= 65535, "attn_tree: %d row blocks of %d heads, %d sequences: more than a grid takes",
              blocks, a.nkv, a.n_seqs);
  e = llg_launch(kernel, dim3(a.n_splits, blocks * a.nkv, a.n_seqs), dim3(THREADS), smem, stream, a);
  if (e != cudaSuccess) return llg_fail("attn_tree: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("attn_tree");
}

template <typename T>
int dispatch(const TreeArgs& a, cudaStream_t stream) {
  const bool few = rows_per_block(a.max_nodes * (a.nh / a.nkv)) == 8;
  if (a.vd <= 64 && a.hd <= 128) return few ? launch<T, 1, 1, 2>(a, stream) : launch<T, 4, 1, 2>(a, stream);
  if (a.vd <= 128 && a.hd <= 128) return few ? launch<T, 1, 2, 2>(a, stream) : launch<T, 4, 2, 2>(a, stream);
  return few ? launch<T, 1, 6, 1>(a, stream) : launch<T, 4, 6, 1>(a, stream);
}

}  // namespace

LLG_API int llg_tree_max_nodes() { return LLG_TREE_NODES; }

// Query rows that a block takes where a tree has up to `rows` of them per key/value head: there are n_seqs * nkv * ceil(rows / this) counters.
LLG_API int llg_attn_tree_rows(int rows) { return rows_per_block(rows); }

// part: [n_seqs * nkv * max_nodes * group][n_splits][vd filled up to 4, + 4] floats where n_splits > 1.
LLG_API int llg_attn_tree_simt(const TreeArgs* args, int dtype, cudaStream_t stream) {
  const TreeArgs& a = *args;
  LLG_REQUIRE(a.nh > 0 && a.nkv > 0 && a.nh % a.nkv == 0, "attn_tree: %d heads are no multiple of %d key/value heads", a.nh, a.nkv);
  LLG_REQUIRE(a.hd > 0 && a.hd <= MAX_HD && a.vd > 0 && a.vd <= MAX_HD, "attn_tree: heads of %d and %d elements (1 to %d)", a.hd, a.vd, MAX_HD);
  LLG_REQUIRE(a.max_nodes > 0 && a.max_nodes <= LLG_TREE_NODES, "attn_tree: trees of up to %d nodes (1 to %d)", a.max_nodes, LLG_TREE_NODES);
  LLG_REQUIRE(a.n_splits >= 1 && (a.n_splits == 1 || (a.part && a.counters)), "attn_tree: %d splits need scratch and counters", a.n_splits);
  LLG_REQUIRE(a.window >= 0 && a.ring_pages > 0 && a.table_width >= a.ring_pages, "attn_tree: bad cache geometry");
  LLG_REQUIRE(a.scale > 0.f, "attn_tree: the softmax scale must be positive");
  if (a.n_seqs <= 0 || a.n_tokens <= 0) return 0;
  if (dtype == LLG_F32) return dispatch<float>(a, stream);
  if (dtype == LLG_BF16) return dispatch<__nv_bfloat16>(a, stream);
  return llg_fail("attn_tree: unknown dtype %d", dtype);
}
