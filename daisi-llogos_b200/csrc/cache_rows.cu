// What becomes of cached rows behind a step: the path of a drafted tree that the logits confirm (tree_accept), the keys of most accumulated
// weight (keep_keys), and the rows that stay, brought together in all layers (move).  No counterpart in the reference, whose speculative
// decoding verifies one chain and only shortens the cache from its end (Inference/SpeculativeDecoder.cs, Inference/KvCache.cs:135).
#include "common.cuh"
#include "cache_args.h"

LLG_API const char* llg_last_error() { return g_llg_error; }

namespace {

// ---- the confirmed path of drafted trees ---------------------------------------------------------------
//
// best_i = argmax of node i's logits (the lowest index of equal ones; NaN is never chosen, 0 where there is nothing else); the path starts at node 0 and goes on to the lowest
// child of the last node whose token is best of the last node; the next token is best of the path's last node.
//
// Reading the logits once is all the time there is: slices of a row over blocks, whose results meet in one 64-bit maximum per row (the
// value's bits in an order that counts upwards, then the index counted downwards: the larger value wins, of equal ones the lower
// index, whatever order blocks come in).  The block that brings a tree's last slice walks it: one warp, two nodes a lane, all in registers.

constexpr int ACC_THREADS = 256;

__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned u = __float_as_uint(v + 0.f);       // -0 counts as 0
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
  return ((unsigned long long)ordered(v) << 32) | (unsigned)(0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// One warp: the path through a tree of n nodes (at most 64); lane i holds nodes i and i + 32.
__device__ __forceinline__ void walk_tree(int n, const int (&token)[2], const int (&parent)[2], const int (&best)[2], int* path, int* n_path,
                                          int* next) {
  const int lane = threadIdx.x & 31;
  int cur = 0, count = 0, mine0 = -1, mine1 = -1, last = -1;
  while (count < n) {
    if (lane == (count & 31)) (count < 32 ? mine0 : mine1) = cur;
    ++count;
    const int b0 = __shfl_sync(0xffffffffu, best[0], cur & 31), b1 = __shfl_sync(0xffffffffu, best[1], cur & 31);
    last = cur < 32 ? b0 : b1;
    const unsigned c0 = __ballot_sync(0xffffffffu, lane < n && lane > cur && parent[0] == cur && token[0] == last);
    const unsigned c1 = __ballot_sync(0xffffffffu, lane + 32 < n && lane + 32 > cur && parent[1] == cur && token[1] == last);
    if (c0) cur = __ffs(c0) - 1;
    else if (c1) cur = __ffs(c1) + 31;
    else break;
  }
  path[lane] = mine0;
  path[lane + 32] = mine1;
  if (lane == 0) {
    *n_path = count;
    *next = last;
  }
}

// A warp: the first of a row's logits that is minus infinity (0: there is none, the row is NaN alone).  Asked where a tree is walked, of the rows that
// hold nothing above: looked for by the blocks that read the row it took 38 registers instead of 32, six blocks a multiprocessor instead of eight, and
// 32 trees' logits 66.9 us instead of 64.4.
__device__ __forceinline__ int first_low(const float* row, int vocab) {
  constexpr int DEEP = 8;                              // asked for at once by a lane
  for (int i0 = 0; i0 < vocab; i0 += 32 * DEEP) {
    int first = 0x7fffffff;
#pragma unroll
    for (int k = DEEP - 1; k >= 0; --k) {
      const int i = i0 + 32 * k + (threadIdx.x & 31);
      if (i < vocab && row[i] == -INFINITY) first = i;
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (first != 0x7fffffff) return first;
  }
  return 0;
}

// rows: n_tokens; slices of `slice` logits per block (blockIdx.x); scratch [n_tokens] maxima, then [n_seqs] counters
template <bool WIDE>
__global__ void __launch_bounds__(ACC_THREADS)
tree_accept_kernel(const float* __restrict__ logits, int vocab, int slice, const int* __restrict__ tokens, const int* __restrict__ parents,
                   const int* __restrict__ cu, int n_seqs, int n_tokens, unsigned long long* __restrict__ scratch, int* __restrict__ path,
                   int* __restrict__ n_path, int* __restrict__ next) {
  __shared__ unsigned long long warp_best[ACC_THREADS / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (row == 0 && blockIdx.x == 0) {                   // trees without a node have nobody else
    for (int b = tid; b < n_seqs; b += ACC_THREADS)
      if (cu[b + 1] <= cu[b]) {
        n_path[b] = 0;
        next[b] = -1;
        for (int i = 0; i < LLG_TREE_NODES; ++i) path[b * LLG_TREE_NODES + i] = -1;
      }
  }
  if (row >= cu[n_seqs]) return;
  int lo = 0, hi = n_seqs - 1;                         // the last tree that starts at or before this row and is not empty
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  const int b = lo, tok0 = cu[b], n = min(cu[b + 1] - tok0, LLG_TREE_NODES);
  if (row - tok0 >= n) return;
  const int v0 = blockIdx.x * slice, v1 = min(vocab, v0 + slice);
  const float* x = logits + (long long)row * vocab;
  float best = -INFINITY;
  int at = v0;
  if (WIDE) {
    const float4* x4 = reinterpret_cast<const float4*>(x);
    int i = v0 / 4 + tid;
    const int end = v1 / 4;
    for (; i + 3 * ACC_THREADS < end; i += 4 * ACC_THREADS) {
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __ldcs(x4 + i + k * ACC_THREADS);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int p = 4 * (i + k * ACC_THREADS);
        if (v[k].x > best) { best = v[k].x; at = p; }
        if (v[k].y > best) { best = v[k].y; at = p + 1; }
        if (v[k].z > best) { best = v[k].z; at = p + 2; }
        if (v[k].w > best) { best = v[k].w; at = p + 3; }
      }
    }
    for (; i < end; i += ACC_THREADS) {
      const float4 v = __ldcs(x4 + i);
      if (v.x > best) { best = v.x; at = 4 * i; }
      if (v.y > best) { best = v.y; at = 4 * i + 1; }
      if (v.z > best) { best = v.z; at = 4 * i + 2; }
      if (v.w > best) { best = v.w; at = 4 * i + 3; }
    }
  } else {
    for (int i = v0 + tid; i < v1; i += ACC_THREADS) {
      const float v = x[i];
      if (v > best) { best = v; at = i; }
    }
  }
  unsigned long long key = warp_max_u64(key_of(best, at));
  if (lane == 0) warp_best[warp] = key;
  __syncthreads();
  if (warp != 0) return;
  key = warp_max_u64(lane < ACC_THREADS / 32 ? warp_best[lane] : 0ull);
  unsigned long long* counter = scratch + n_tokens + b;
  unsigned long long ticket = 0;
  if (lane == 0) {
    atomicMax(scratch + row, key);
    __threadfence();
    ticket = atomicAdd(counter, 1ull);
  }
  ticket = __shfl_sync(0xffffffffu, ticket, 0);
  if (ticket != (unsigned long long)n * gridDim.x - 1) return;
  __threadfence();
  int token[2], parent[2], top[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = lane + 32 * e;
    const bool there = i < n;
    token[e] = there ? tokens[tok0 + i] : -1;
    parent[e] = there ? parents[tok0 + i] : -1;
    top[e] = -1;
    bool none = false;                                 // nothing above minus infinity in the node's row: its first place may be NaN
    if (there) {
      const unsigned long long most = __ldcg(scratch + tok0 + i);
      top[e] = (int)(0xffffffffu - (unsigned)most);
      none = (unsigned)(most >> 32) == ordered(-INFINITY);
      scratch[tok0 + i] = 0;
    }
    for (unsigned rows = __ballot_sync(0xffffffffu, none); rows; rows &= rows - 1) {
      const int r = __ffs(rows) - 1, first = first_low(logits + (long long)(tok0 + 32 * e + r) * vocab, vocab);
      if (lane == r) top[e] = first;
    }
  }
  if (lane == 0) *counter = 0;
  walk_tree(n, token, parent, top, path + (long long)b * LLG_TREE_NODES, n_path + b, next + b);
}

// The same with the nodes' tokens already picked; one warp per tree.
__global__ void __launch_bounds__(128)
tree_walk_kernel(const int* __restrict__ picked, const int* __restrict__ tokens, const int* __restrict__ parents, const int* __restrict__ cu,
                 int n_seqs, int* __restrict__ path, int* __restrict__ n_path, int* __restrict__ next) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= n_seqs) return;
  const int tok0 = cu[b], n = max(0, min(cu[b + 1] - tok0, LLG_TREE_NODES));
  int token[2], parent[2], top[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = lane + 32 * e;
    const bool there = i < n;
    token[e] = there ? tokens[tok0 + i] : -1;
    parent[e] = there ? parents[tok0 + i] : -1;
    top[e] = there ? picked[tok0 + i] : -1;
  }
  walk_tree(n, token, parent, top, path + (long long)b * LLG_TREE_NODES, n_path + b, next + b);
}

// ---- the keys of most weight ----------------------------------------------------------------------------
//
// Of a sequence's `len` positions in a layer and head, `keep` stay: the first `first`, the newest `recent`, and of those between them the ones of
// most weight (of equal ones the lower position; NaN counts as less than everything), written in ascending order.
//
// A block takes one (layer, sequence, head) and keeps its weights in registers, so that they are read once.  They are compared as whole numbers in
// the floats' order.  The weight of rank `need` is found by counting: the range between the least and the largest is cut into 2,048 bins (of
// equal width in that order, which is the floats' logarithm, so weights spread over the bins), the counts are added up from the top to the
// bin that holds the rank, and that bin is the next range; once at most a block's number of weights is left they are ranked directly.  (A
// bisection over the 32 bits, a bit and a block's count a round, was bound by its instructions: 131 us for eight sequences of 5,000 to
// 8,190 keys, 32 layers, 8 heads.)  A warp holds a run of neighbouring positions, so that ballots give every chosen position its place in
// ascending order with one sum over the warps.

constexpr int KEEP_THREADS = 512, KEEP_WARPS = KEEP_THREADS / 32, KEEP_BINS = 2048;
static_assert(KEEP_BINS == 4 * KEEP_THREADS, "a thread clears and adds up four bins");

__device__ __forceinline__ unsigned weight_key(float w) { return w != w ? 1u : ordered(w); }      // the least number's is 0x007fffff

// VPL: weights that a lane keeps in registers (0: read again every time)
template <int VPL>
__global__ void __launch_bounds__(KEEP_THREADS, VPL <= 16 ? 4 : 2)
keep_keys_kernel(const float* __restrict__ weights, long long layer_stride, int width, int nkv, const int* __restrict__ slots,
                 const int* __restrict__ lengths, const int* __restrict__ keeps, int first, int recent, int* __restrict__ chosen, int most,
                 int max_len) {
  __shared__ int count_of[KEEP_WARPS], place_of[KEEP_WARPS], tie_of[KEEP_WARPS];
  __shared__ __align__(16) int bins[KEEP_BINS];
  __shared__ unsigned least_of[KEEP_WARPS], most_of[KEEP_WARPS], left[KEEP_THREADS], found;
  __shared__ int bin_at, bin_above, n_left;
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = min(lengths[b], max_len), keep = min(min(keeps[b], len), most);
  if (keep <= 0) return;
  int* out = chosen + (((long long)layer * gridDim.y + b) * nkv + h) * most;
  const int f_end = min(first, len), r_begin = max(f_end, len - recent);      // [0, f_end) and [r_begin, len) stay
  const int between = r_begin - f_end;
  int need = keep - f_end - (len - r_begin);                                  // of those between
  for (int j = tid; j < min(f_end, keep); j += KEEP_THREADS) out[j] = j;
  for (int j = max(0, need) + f_end + tid; j < keep; j += KEEP_THREADS) out[j] = r_begin + j - f_end - max(0, need);
  if (need <= 0) return;
  const float* w = weights + layer * layer_stride + ((long long)slots[b] * nkv + h) * width + f_end;
  out += f_end;
  const int per_lane = VPL ? VPL : (between + KEEP_THREADS - 1) / KEEP_THREADS, run = per_lane * 32;
  const int p0 = warp * run + lane;                                           // this lane's positions between: p0, p0 + 32, ...
  auto fetch = [&](int i) -> unsigned { return p0 + 32 * i < between ? weight_key(w[p0 + 32 * i]) : 0u; };      // 0: not there
  unsigned v[VPL ? VPL : 1];
  if (VPL) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = fetch(i);
  }
  auto value = [&](int i) -> unsigned { return VPL ? v[i] : fetch(i); };
  const int all_needed = need;
  // the weight of rank `need`
  unsigned threshold = 1u;
  if (need < between) {
    unsigned lo = 0xffffffffu, hi = 0u;                                       // (the least less one)
#pragma unroll
    for (int i = 0; i < (VPL ? VPL : per_lane); ++i) {
      const unsigned x = value(i);
      lo = min(lo, x - 1u);                                                   // (what is not there: the largest number)
      hi = max(hi, x);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      least_of[warp] = lo;
      most_of[warp] = hi;
    }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, lane < KEEP_WARPS ? least_of[lane] : 0xffffffffu) + 1u;
    hi = __reduce_max_sync(0xffffffffu, lane < KEEP_WARPS ? most_of[lane] : 0u);
    for (;;) {
      const int shift = max(0, 32 - __clz(hi - lo) - 11);                     // (hi - lo) >> shift < KEEP_BINS; lo and hi are the block's
      reinterpret_cast<int4*>(bins)[tid] = make_int4(0, 0, 0, 0);
      if (tid == 0) n_left = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < (VPL ? VPL : per_lane); ++i) {
        const unsigned x = value(i) - lo;
        if (x <= hi - lo) atomicAdd(&bins[x >> shift], 1);
      }
      __syncthreads();
      // a thread's four bins, counted from the top: how many weights lie above them
      const int4 mine = reinterpret_cast<int4*>(bins)[KEEP_THREADS - 1 - tid];
      const int here = mine.x + mine.y + mine.z + mine.w;
      int upto = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      if (lane == 31) count_of[warp] = upto;
      __syncthreads();
      const int before = lane < warp ? count_of[lane] : 0;
      int above = upto - here + __reduce_add_sync(0xffffffffu, before);
      if (above < need && need <= above + here) {                             // one thread
        const int four[4] = {mine.w, mine.z, mine.y, mine.x};
        int k = 0;
        while (above + four[k] < need) above += four[k++];
        bin_at = (KEEP_THREADS - 1 - tid) * 4 + 3 - k;
        bin_above = above;
      }
      __syncthreads();
      const int count = bins[bin_at];
      need -= bin_above;
      lo += (unsigned)bin_at << shift;
      hi = shift == 0 ? lo : min(hi, lo + ((1u << shift) - 1u));
      if (lo == hi) {
        threshold = lo;
        break;
      }
      if (count <= KEEP_THREADS) {
#pragma unroll
        for (int i = 0; i < (VPL ? VPL : per_lane); ++i) {
          const unsigned x = value(i);
          if (x - lo <= hi - lo) left[atomicAdd(&n_left, 1)] = x;
        }
        __syncthreads();
        if (tid < count) {
          const unsigned x = left[tid];
          int more = 0, same = 0;
          for (int k = 0; k < count; ++k) {
            more += (int)(left[k] > x);
            same += (int)(left[k] == x);
          }
          if (more < need && need <= more + same) found = x;                  // all that do have this weight
        }
        __syncthreads();
        threshold = found;
        break;
      }
      __syncthreads();                                                        // bins and bin_at have been read
    }
  }
  // how many reach the threshold: exactly as many as are needed where all of that very weight stay
  int reach = 0;
#pragma unroll
  for (int i = 0; i < (VPL ? VPL : per_lane); ++i) reach += (int)(value(i) >= threshold);
  reach = __reduce_add_sync(0xffffffffu, reach);
  if (lane == 0) place_of[warp] = reach;
  __syncthreads();
  const int theirs = lane < KEEP_WARPS ? place_of[lane] : 0;
  int at = __reduce_add_sync(0xffffffffu, lane < warp ? theirs : 0);
  const unsigned below = (1u << lane) - 1u;
  if (__reduce_add_sync(0xffffffffu, theirs) == all_needed) {
#pragma unroll
    for (int i = 0; i < (VPL ? VPL : per_lane); ++i) {
      const bool mine = value(i) >= threshold;
      const unsigned taken = __ballot_sync(0xffffffffu, mine);
      if (mine) out[at + __popc(taken & below)] = f_end + p0 + 32 * i;
      at += __popc(taken);
    }
    return;
  }
  // of those of that very weight the lowest positions
  int ties = 0;
  for (int i = 0; i < per_lane; ++i) ties += (int)(fetch(i) == threshold);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) tie_of[warp] = ties;
  __syncthreads();
  int all_ties = 0, all = 0, ties_before = 0;
  for (int k = 0; k < KEEP_WARPS; ++k) {
    all += place_of[k];
    all_ties += tie_of[k];
    if (k < warp) ties_before += tie_of[k];
  }
  const int room = all_needed - (all - all_ties);                             // for ties
  at += min(ties_before, room) - ties_before;
  int ties_left = max(0, room - ties_before);
  for (int i = 0; i < per_lane; ++i) {
    const unsigned x = fetch(i);
    const unsigned tie = __ballot_sync(0xffffffffu, x == threshold);
    const bool mine = x > threshold || (x == threshold && __popc(tie & below) < ties_left);
    const unsigned taken = __ballot_sync(0xffffffffu, mine);
    if (mine) out[at + __popc(taken & below)] = f_end + p0 + 32 * i;
    at += __popc(taken);
    ties_left = max(0, ties_left - __popc(tie));
  }
}

// ---- rows to new places ----------------------------------------------------------------------------------
//
// A block takes the key (or value) rows of one layer, sequence and head, a batch of rows after the other: all of a batch are read before the first
// is written.  Sources ascend and none lies before its target, so what a batch writes no later batch reads, and the move needs no copy.
// Such a list cannot be shared by blocks, and its time is the chain of its batches (source, page, row, write), so the launch takes blocks as large
// as let all lists run at once: a second wave of few blocks would move the last rows at the speed of their latency.  The next batch's sources
// are asked for before this one is written, and all that a block begins with is asked for at once.

constexpr int MOVE_DEEP = 4, MOVE_MAX_THREADS = 1024;

template <typename U>
__device__ __forceinline__ void move_rows(const MoveArgs& a, U* pool, int units, int b, int h, const int* src) {
  const int tid = threadIdx.x, side = blockDim.x / units, rows = side * MOVE_DEEP;      // rows that the block reads side by side, and of a batch
  const int r0 = tid / units, u = tid - r0 * units;                            // this thread's first row of a batch, and its unit of a row
  const bool works = r0 < side;
  int s[MOVE_DEEP];
#pragma unroll
  for (int k = 0; k < MOVE_DEEP; ++k) s[k] = works && r0 + k * side < a.most ? src[r0 + k * side] : -1;
  const int slot = a.slots[b], count = min(a.count[b], a.most), base = a.base[b];
  const int* table = a.page_table + (long long)slot * a.table_width;
  pool += (long long)h * LLG_PAGE * units + u;
  const unsigned page_units = (unsigned)a.nkv * LLG_PAGE * units;
  auto place = [&](int pos) -> U* {
    unsigned lp = (unsigned)pos / LLG_PAGE;
    if (lp >= (unsigned)a.ring_pages) lp %= (unsigned)a.ring_pages;
    return pool + (long long)((unsigned)table[lp] * (unsigned long long)page_units + ((unsigned)pos % LLG_PAGE) * (unsigned)units);
  };
  for (int j0 = 0; j0 < count; j0 += rows) {
    U v[MOVE_DEEP];
    bool goes[MOVE_DEEP];
#pragma unroll
    for (int k = 0; k < MOVE_DEEP; ++k) {
      const int j = j0 + r0 + k * side;
      goes[k] = works && j < count && s[k] > j;                               // a row that stays where it is costs nothing
      if (goes[k]) v[k] = *place(base + s[k]);
    }
#pragma unroll
    for (int k = 0; k < MOVE_DEEP; ++k) {
      const int j = j0 + rows + r0 + k * side;
      s[k] = works && j < count ? src[j] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MOVE_DEEP; ++k)
      if (goes[k]) *place(base + j0 + r0 + k * side) = v[k];
  }
}

__global__ void __launch_bounds__(MOVE_MAX_THREADS, 2) move_rows_kernel(MoveArgs a) {
  const int h = blockIdx.x, b = blockIdx.y;
  const int per_layer = a.pools_per_layer + (a.weights ? 1 : 0);
  const int layer = blockIdx.z / per_layer, which = blockIdx.z - layer * per_layer;
  const int* src = a.source + layer * a.source_layer + b * a.source_seq + h * a.source_head;
  if (which == a.pools_per_layer) {
    // the weights of the keys that stay, moved along
    const int count = min(a.count[b], a.most), base = a.base[b], threads = blockDim.x;
    float* w = a.weights + layer * a.weight_layer + ((long long)a.slots[b] * a.nkv + h) * a.weight_width;
    for (int j0 = 0; j0 < count; j0 += threads) {
      const int j = j0 + threadIdx.x;
      const int s = j < count ? src[j] : 0;
      const bool goes = j < count && s > j && base + s < a.weight_width;
      const float v = goes ? w[base + s] : 0.f;
      __syncthreads();
      if (goes) w[base + j] = v;
    }
    return;
  }
  void* pool = a.pools[layer * a.pools_per_layer + which];
  const int bytes = which == 0 ? a.row_bytes[0] : a.row_bytes[1];
  if (bytes % 16 == 0) move_rows<uint4>(a, (uint4*)pool, bytes / 16, b, h, src);
  else if (bytes % 4 == 0) move_rows<unsigned>(a, (unsigned*)pool, bytes / 4, b, h, src);
  else move_rows<unsigned short>(a, (unsigned short*)pool, bytes / 2, b, h, src);
}

}  // namespace

// Blocks' slices of a row of logits: enough of them that few rows still fill the GPU, none shorter than a block reads in one turn.
static int accept_slice(int n_tokens, int vocab) {
  const long long blocks = 8LL * llg_sm_count();
  long long slice = ((long long)n_tokens * vocab + blocks - 1) / blocks;
  const int turn = ACC_THREADS * 16;
  slice = (slice + turn - 1) / turn * turn;
  return (int)(slice > 16 * turn ? 16 * turn : slice);
}

LLG_API int llg_tree_accept(const float* logits, int vocab, const int* tokens, const int* parents, const int* cu, int n_seqs, int n_tokens,
                            unsigned long long* scratch, int* path, int* n_path, int* next, cudaStream_t stream) {
  LLG_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && vocab > 0, "tree_accept: bad sizes");
  LLG_REQUIRE(n_tokens <= 65535, "tree_accept: %d nodes in one call are more than a grid takes (65535)", n_tokens);
  LLG_REQUIRE(scratch, "tree_accept: needs scratch");
  if (n_seqs == 0) return 0;
  if (n_tokens == 0) return llg_fail("tree_accept: trees without any node");
  const int slice = accept_slice(n_tokens, vocab);
  const dim3 grid((vocab + slice - 1) / slice, n_tokens);
  const bool wide = vocab % 4 == 0 && (uintptr_t)logits % 16 == 0;
  cudaError_t e = llg_launch(wide ? tree_accept_kernel<true> : tree_accept_kernel<false>, grid, dim3(ACC_THREADS), 0, stream, logits, vocab, slice,
                             tokens, parents, cu, n_seqs, n_tokens, scratch, path, n_path, next);
  if (e != cudaSuccess) return llg_fail("tree_accept: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("tree_accept");
}

LLG_API int llg_tree_walk(const int* picked, const int* tokens, const int* parents, const int* cu, int n_seqs, int* path, int* n_path, int* next,
                          cudaStream_t stream) {
  LLG_REQUIRE(n_seqs >= 0, "tree_accept: bad sizes");
  if (n_seqs == 0) return 0;
  cudaError_t e = llg_launch(tree_walk_kernel, dim3((n_seqs + 3) / 4), dim3(128), 0, stream, picked, tokens, parents, cu, n_seqs, path, n_path, next);
  if (e != cudaSuccess) return llg_fail("tree_accept: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("tree_accept");
}

// weights [layers][slots][nkv][width] (layer_stride elements a layer), chosen [layers][n_seqs][nkv][most]; max_len bounds the lengths
LLG_API int llg_keep_keys(const float* weights, long long layer_stride, int width, int nkv, int n_layers, int n_seqs, const int* slots,
                          const int* lengths, const int* keeps, int first, int recent, int* chosen, int most, int max_len,
                          cudaStream_t stream) {
  LLG_REQUIRE(max_len >= 0 && max_len <= width, "keep_keys: sequences of up to %d keys in rows of %d weights", max_len, width);
  LLG_REQUIRE(width > 0 && nkv > 0 && n_layers >= 0 && n_seqs >= 0 && most >= 0, "keep_keys: bad sizes");
  LLG_REQUIRE(first >= 0 && recent >= 0, "keep_keys: first %d and recent %d must not be negative", first, recent);
  LLG_REQUIRE(n_seqs <= 65535 && n_layers <= 65535, "keep_keys: %d sequences, %d layers: more than a grid takes", n_seqs, n_layers);
  if (n_layers == 0 || n_seqs == 0 || most == 0) return 0;
  const dim3 grid(nkv, n_seqs, n_layers);
  auto kernel = max_len <= KEEP_THREADS * 4 ? keep_keys_kernel<4> : max_len <= KEEP_THREADS * 16 ? keep_keys_kernel<16>
              : max_len <= KEEP_THREADS * 32 ? keep_keys_kernel<32> : keep_keys_kernel<0>;
  cudaError_t e = llg_launch(kernel, grid, dim3(KEEP_THREADS), 0, stream, weights, layer_stride, width, nkv, slots, lengths, keeps, first, recent,
                             chosen, most, max_len);
  if (e != cudaSuccess) return llg_fail("keep_keys: launch: %s", cudaGetErrorString(e));
  return llg_check_launch("keep_keys");
}

// The next kernel starts when this one has ended: attention looks at pages before its own wait.
LLG_API int llg_move_rows(const MoveArgs* args, cudaStream_t stream) {
  const MoveArgs& a = *args;
  LLG_REQUIRE(a.n_layers >= 0 && a.n_seqs >= 0 && a.nkv > 0 && a.pools_per_layer >= 1 && a.pools_per_layer <= 2, "move: bad sizes");
  LLG_REQUIRE(a.ring_pages > 0 && a.table_width >= a.ring_pages, "move: bad cache geometry");
  int units = 1;
  for (int i = 0; i < a.pools_per_layer; ++i) {
    LLG_REQUIRE(a.row_bytes[i] > 0 && a.row_bytes[i] % 2 == 0, "move: rows of %d bytes", a.row_bytes[i]);
    const int u = a.row_bytes[i] / (a.row_bytes[i] % 16 == 0 ? 16 : a.row_bytes[i] % 4 == 0 ? 4 : 2);
    units = u > units ? u : units;
  }
  LLG_REQUIRE(units <= MOVE_MAX_THREADS, "move: rows of %d and %d bytes", a.row_bytes[0], a.row_bytes[1]);
  const long long z = (long long)a.n_layers * (a.pools_per_layer + (a.weights ? 1 : 0));
  LLG_REQUIRE(a.n_seqs <= 65535 && z <= 65535, "move: %d sequences, %d layers: more than a grid takes", a.n_seqs, a.n_layers);
  if (z == 0 || a.n_seqs == 0 || a.most <= 0) return 0;
  // as many threads a block as let all lists run at once (2,048 threads a multiprocessor), no more than a list has work for, and a row's at least
  const long long lists = z * a.n_seqs * a.nkv, fit = 2048LL * llg_sm_count() / lists, work = (long long)a.most * units;
  int threads = 128;
  while (threads < MOVE_MAX_THREADS && (threads < units || (2 * threads <= fit && threads * MOVE_DEEP < work))) threads *= 2;
  move_rows_kernel<<<dim3(a.nkv, a.n_seqs, (unsigned)z), threads, 0, stream>>>(a);
  return llg_check_launch("move");
}
