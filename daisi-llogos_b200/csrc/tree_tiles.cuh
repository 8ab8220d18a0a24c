// What the tensor-core kernels for drafted trees share (attention_tree_mma.cu, attention_tree_tc.cu): barriers with limits, TMA boxes of cache pages,
// the softmax's arithmetic, and the list of work that blocks cut into runs.
#pragma once
#include "common.cuh"
#include "cache_args.h"

#include <cuda.h>

#include <mutex>

namespace {

typedef __nv_bfloat16 bf16;
constexpr int TK = 64;                       // keys per tile = one cache page
constexpr int MAX_SEQS = 1024;               // sequences whose work fits the plan in shared memory
constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// false when the limit ran out or another role of the block gave up
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  int spins = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++spins & 1023) == 0) {
      if (*abort_flag) return false;
      if (now_ns() - t0 > WAIT_LIMIT_NS) return false;
    }
  }
  return true;
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// x: first element of the box along the head dimension (0 or 64: a multiple of 8 elements, 16 bytes), y: first row
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// 2^x by the special-function unit alone; arguments are <= 0 or -inf, or bounded by the caller.  (Somewhat less exact than
// exp2f: key weights of a decode step are off by 4.5e-7 of the largest, a plain form in 32 bits by 3.1e-7.)
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^d for a whole number d <= 0 (or -inf), exactly
__device__ __forceinline__ float pow2_whole(float d) {
  return d < -126.f ? 0.f : __int_as_float((127 + (int)d) << 23);
}
// whether one of two packed bfloat16 numbers is infinite or NaN
__device__ __forceinline__ bool not_finite(uint32_t x) {
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// A sequence's tree: its nodes, cached keys, and the key tiles that its rows look at.
struct TreeShape {
  int tok0, n, lb, slot, t_first, tiles;
};

// The work of a launch is one list: sequence by sequence, key/value head by key/value head, row block by row block, key tile by key tile.
// Blocks cut it into equal runs.  Every block works the list out itself, in shared memory: per sequence the units, the row blocks and the weight of
// one head in the sequences before it, and what there is to know of the first STAGED sequences.  (Counts are 32-bit: a division of 64
// bits takes a hundred instructions, and a block's begin is a chain of them; calls whose list is longer go to another kernel, see list_fits.)
constexpr int STAGED = 128;
struct Plan {
  int sums[MAX_SEQS + 1], blocks[MAX_SEQS + 1];
  int4 seq[STAGED];                                // tok0, n, lb, slot
  int3 warp_total[32];
};

__device__ __forceinline__ TreeShape shape_of(const TreeArgs& a, int4 q) {
  TreeShape s;
  s.tok0 = q.x;
  s.n = q.y;
  s.lb = q.z;
  s.slot = q.w;
  // no row sees less than this under a window (a row without any bit stands one place before the root)
  s.t_first = a.window > 0 ? max(0, s.lb - a.window) / TK : 0;
  s.tiles = s.n > 0 ? (s.lb + s.n + TK - 1) / TK - s.t_first : 0;
  return s;
}
__device__ __forceinline__ int4 fetch_seq(const TreeArgs& a, int b) {
  const int t0 = a.cu_tokens[b], t1 = a.cu_tokens[b + 1], lb = a.len_before[b], slot = a.slots[b];
  return make_int4(t0, max(0, min(min(t1, a.n_tokens) - t0, a.max_nodes)), lb, slot);
}
__device__ __forceinline__ TreeShape tree_shape(const TreeArgs& a, const Plan& p, int b) {
  return shape_of(a, b < STAGED ? p.seq[b] : fetch_seq(a, b));
}

struct Unit {
  int b, kvh, rb, t;
};
__device__ __forceinline__ Unit locate(const Plan& p, int n_seqs, int nkv, int u) {
  int lo = 0, hi = n_seqs - 1;                     // last b with nkv * sums[b] <= u
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (nkv * p.sums[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  Unit c;
  c.b = lo;
  const unsigned rbs = p.blocks[lo + 1] - p.blocks[lo], tiles = (unsigned)(p.sums[lo + 1] - p.sums[lo]) / rbs;
  const unsigned r = u - nkv * p.sums[lo], pair = r / tiles;
  c.t = r - pair * tiles;
  c.kvh = pair / rbs;
  c.rb = pair - c.kvh * rbs;
  return c;
}

// All threads of a block: the plan for row blocks of `rows` query rows, and (weights not null) what `weight(rows, row blocks, tiles)` gives a head.
template <int THREADS, typename Weight>
__device__ __forceinline__ void plan_units(const TreeArgs& a, int rows, Plan& p, int* weights, Weight weight) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.nh / a.nkv;
  const int per = (a.n_seqs + THREADS - 1) / THREADS;
  const int b0 = tid * per, b1 = min(a.n_seqs, b0 + per);
  int units = 0, rbs = 0, ws = 0;
  int4 only = make_int4(0, 0, 0, 0);               // of a thread with one sequence
  auto add = [&](int4 q) {
    const TreeShape s = shape_of(a, q);
    const int r = (unsigned)(s.n * G + rows - 1) / (unsigned)rows;
    units += r * s.tiles;
    rbs += r;
    ws += weight(s.n * G, r, s.tiles);
  };
  for (int b = b0; b < b1; ++b) {
    only = fetch_seq(a, b);
    if (b < STAGED) p.seq[b] = only;
    add(only);
  }
  int iu = units, ir = rbs, iw = ws;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pu = __shfl_up_sync(0xffffffffu, iu, o), pr = __shfl_up_sync(0xffffffffu, ir, o), pw = __shfl_up_sync(0xffffffffu, iw, o);
    if (lane >= o) {
      iu += pu;
      ir += pr;
      iw += pw;
    }
  }
  if (lane == 31) p.warp_total[warp] = make_int3(iu, ir, iw);
  __syncthreads();
  int before_u = iu - units, before_r = ir - rbs, before_w = iw - ws;
  for (int w = 0; w < warp; ++w) {
    before_u += p.warp_total[w].x;
    before_r += p.warp_total[w].y;
    before_w += p.warp_total[w].z;
  }
  if (tid == 0) {
    p.sums[0] = p.blocks[0] = 0;
    if (weights) weights[0] = 0;
  }
  units = before_u;
  rbs = before_r;
  ws = before_w;
  for (int b = b0; b < b1; ++b) {
    add(per == 1 ? only : fetch_seq(a, b));
    p.sums[b + 1] = units;
    p.blocks[b + 1] = rbs;
    if (weights) weights[b + 1] = ws;
  }
  __syncthreads();
}

// ---- joining runs that share rows -----------------------------------------------------------------------
//
// A run that ends inside a (sequence, head, row block), or begins inside one, leaves that segment as partial rows.  Only a run's first and last
// segment can be such, so a block has two places for them: one for a segment that begins the run, one for a segment that ends it and does
// not begin it.  A place holds the sums column by column ([HDP / 4][ROWS] of four columns each, so that threads with neighbouring rows write and
// read neighbouring addresses), then every row's maximum and sum of weights.  Every block leaves one note: the segment that it begins and that
// others go on with, if there is one.  A second kernel, a thread per row and 16 columns, joins what a note tells of in the runs' order.  (Joined by
// the block that finished last, eight trees behind 8,190 keys took 12 us longer: one multiprocessor then read all of a pair's partial rows.)
struct Note {
  int parts, place, n_rows, row0, tok0, kvh, pad[2];      // parts 0: nothing; place: the first part's; the others lie at the beginning of their blocks' runs
};

template <int HDP, int ROWS>
struct Place {
  static constexpr long long FLOATS = (long long)ROWS * (HDP + 2);
  __device__ static float4* sums(float* part, int place) { return reinterpret_cast<float4*>(part + place * FLOATS); }
  __device__ static float2* ends(float* part, int place) { return reinterpret_cast<float2*>(part + place * FLOATS + (long long)ROWS * HDP); }
  __host__ __device__ static long long floats(int blocks) { return 2 * blocks * FLOATS + blocks * (long long)(sizeof(Note) / 4); }
  __device__ static Note* notes(float* part, int blocks) { return reinterpret_cast<Note*>(part + 2 * blocks * FLOATS); }
};

constexpr int JOIN_THREADS = 128, JOIN_COLS = 16;

template <int HDP, int ROWS>
__global__ void __launch_bounds__(JOIN_THREADS) tree_join_kernel(TreeArgs a, int blocks) {
  typedef Place<HDP, ROWS> P;
  pdl_launch_dependents();
  pdl_wait();
  const Note n = P::notes(a.part, blocks)[blockIdx.x];
  if (n.parts <= 1) return;
  const int item = blockIdx.y * JOIN_THREADS + threadIdx.x, row = item % ROWS, d0 = item / ROWS * JOIN_COLS;
  if (row >= n.n_rows || d0 >= a.vd) return;
  float M = -INFINITY, L = 0.f;
  float4 acc[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int DEEP = 4;                                 // parts asked for at once
  for (int k0 = 0; k0 < n.parts; k0 += DEEP) {
    float2 ml[DEEP];
    float4 v[DEEP][4];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      const bool there = k0 + k < n.parts;
      const int place = k0 + k == 0 ? n.place : 2 * (n.place / 2 + k0 + k);
      ml[k] = there ? __ldcg(P::ends(a.part, place) + row) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        v[k][q] = there ? __ldcg(P::sums(a.part, place) + (d0 / 4 + q) * ROWS + row) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = M;
#pragma unroll
    for (int k = 0; k < DEEP; ++k) top = fmaxf(top, ml[k].x);
    const float f = M == -INFINITY ? 0.f : pow2_whole(M - top);
    M = top;
    L *= f;
#pragma unroll
    for (int q = 0; q < 4; ++q) { acc[q].x *= f; acc[q].y *= f; acc[q].z *= f; acc[q].w *= f; }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      if (ml[k].x == -INFINITY) continue;                 // a part in which the row sees nothing
      const float w = pow2_whole(ml[k].x - M);
      L += w * ml[k].y;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        acc[q].x += w * v[k][q].x;
        acc[q].y += w * v[k][q].y;
        acc[q].z += w * v[k][q].z;
        acc[q].w += w * v[k][q].w;
      }
    }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  const int G = a.nh / a.nkv, node = (n.row0 + row) / G, head = n.kvh * G + (n.row0 + row) - node * G;
  bf16* dst = (bf16*)a.out + ((long long)(n.tok0 + node) * a.nh + head) * a.vd + d0;
#pragma unroll
  for (int q = 0; q < 4; q += 2) {
    if (d0 + 4 * q < a.vd)                                // (value sizes are multiples of 8)
      *reinterpret_cast<uint4*>(dst + 4 * q) = make_uint4(pack_bf16(acc[q].x * inv, acc[q].y * inv), pack_bf16(acc[q].z * inv, acc[q].w * inv),
                                                          pack_bf16(acc[q + 1].x * inv, acc[q + 1].y * inv), pack_bf16(acc[q + 1].z * inv, acc[q + 1].w * inv));
  }
}

template <int HDP, int ROWS>
inline int launch_join(const TreeArgs& a, int blocks, const char* what, cudaStream_t stream) {
  cudaError_t e = llg_launch(tree_join_kernel<HDP, ROWS>, dim3(blocks, (ROWS * (HDP / JOIN_COLS) + JOIN_THREADS - 1) / JOIN_THREADS), dim3(JOIN_THREADS), 0,
                             stream, a, blocks);
  if (e != cudaSuccess) return llg_fail("%s: launch: %s", what, cudaGetErrorString(e));
  return llg_check_launch(what);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}

// Boxes of 64 rows x 64 head dimensions (128 bytes, swizzled) out of the pages seen as [pages x kv heads x 64][hd]; what lies behind hd reads as 0.
inline bool page_map(const void* base, long long rows, int hd, CUtensorMap* result) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint32_t estr[2] = {1, 1};
  cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)TK};
  return fn(result, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether a launch's list of work, `per_tile` for each key tile of a row block and `per_block` for each row block, fits the kernels' 32-bit counts if
// every sequence is as long as it may be (a block's end lies up to a run behind the list's: a million blocks' worth of room).
inline bool list_fits(long long n_seqs, long long nkv, long long row_blocks, long long max_len, long long per_tile, long long per_block) {
  return (per_tile * ((max_len + TK - 1) / TK) + per_block) * row_blocks < ((1LL << 31) - (1LL << 20)) / (nkv * n_seqs);
}

// What a launch wants of its arguments.
inline int check_tree(const TreeArgs& a, const char* what) {
  LLG_REQUIRE(a.nh > 0 && a.nkv > 0 && a.nh % a.nkv == 0, "%s: %d heads are no multiple of %d key/value heads", what, a.nh, a.nkv);
  LLG_REQUIRE(a.max_nodes > 0 && a.max_nodes <= LLG_TREE_NODES, "%s: trees of up to %d nodes (1 to %d)", what, a.max_nodes, LLG_TREE_NODES);
  LLG_REQUIRE(a.n_seqs <= MAX_SEQS, "%s: %d sequences (at most %d)", what, a.n_seqs, MAX_SEQS);
  LLG_REQUIRE(a.window >= 0 && a.ring_pages > 0 && a.table_width >= a.ring_pages, "%s: bad cache geometry", what);
  LLG_REQUIRE(a.scale > 0.f, "%s: the softmax scale must be positive", what);
  LLG_REQUIRE(a.part && a.max_len > 0 && a.n_pages > 0, "%s: needs scratch, a bound on the lengths and pages", what);
  LLG_REQUIRE((uintptr_t)a.k_pages % 16 == 0 && (uintptr_t)a.v_pages % 16 == 0 && (uintptr_t)a.q % 16 == 0, "%s: storage must be 16-byte aligned", what);
  LLG_REQUIRE((long long)a.n_pages * a.nkv * TK < 2147483647LL, "%s: too many page rows for a tensor map coordinate", what);
  return 0;
}

}  // namespace
