// Argument structures of the kernels for drafted trees and shortened caches, shared by the libraries and Python (ctypes mirrors).
#pragma once

// Most nodes of a drafted tree: a node's ancestors are the bits of one 64-bit word, and a tree is as wide as one cache page.
#define LLG_TREE_NODES 64

// Attention of drafted trees over the paged cache (attention_tree.cu, attention_tree_mma.cu).  Sequence b holds len_before[b] keys; its nodes
// are the packed tokens cu_tokens[b] .. cu_tokens[b + 1], at most max_nodes (64), whose keys and values lie in the pages at positions
// len_before[b] + i.  With depth_i = (bits of ancestors[i]) - 1, node i sees the cached positions p < len_before (under a window p > len_before
// + depth_i - window) and the nodes j of its tree whose bit is set in ancestors[i] (under a window depth_i - depth_j < window).
struct TreeArgs {
  const void* q;              // [n_tokens][nh][hd]
  const void* k_pages;        // [n_pages][nkv][LLG_PAGE][hd]
  const void* v_pages;        // [n_pages][nkv][LLG_PAGE][vd]
  const int* page_table;      // [slots][table_width]
  int table_width, ring_pages;
  const int* slots;           // [n_seqs]
  const int* cu_tokens;       // [n_seqs + 1]
  const int* len_before;      // [n_seqs]
  const long long* ancestors; // [n_tokens]
  void* out;                  // [n_tokens][nh * vd]
  float* part;                // partial results; see the kernels
  int* counters;              // zero before and after a launch
  int n_seqs, n_tokens, max_nodes, n_pages, nh, nkv, hd, vd, n_splits, max_len;
  float scale;
  int window;
};

// What the last `last` queries of every sequence of a step give each key (key_weights.cu).
struct KeyWeightArgs {
  const void* q;              // [n_tokens][nh][hd]
  const void* k_pages;        // [n_pages][nkv][LLG_PAGE][hd]
  const int* page_table;      // [slots][table_width]
  int table_width;
  const int* slots;           // [n_seqs]
  const int* cu_tokens;       // [n_seqs + 1]
  const int* len_before;      // [n_seqs]
  float* weights;             // [slots][nkv][weight_width]
  int weight_width;
  float* stats;               // [n_seqs][nkv][splits][rows][2], rows = nh / nkv * last: a split's maximum and sum
  float* scores;              // [n_seqs][nkv][rows][splits * split_keys], or null: the second pass works them out again
  int n_seqs, n_tokens, nh, nkv, hd, last, splits, split_keys;
  float scale;
};


// Rows of a paged cache brought to new places in all layers (cache_rows.cu).  For layer l, sequence b and key/value head h, the row of
// position base[b] + source[l][b][h][j] goes to position base[b] + j, j < count[b]; source ascends and source[j] >= j.
struct MoveArgs {
  void* const* pools;         // [layers][pools_per_layer]: key pages, value pages
  int n_layers, pools_per_layer;
  int row_bytes[2];           // of a key row and a value row
  const int* page_table;
  int table_width, ring_pages;
  const int* slots;
  const int* base;
  const int* source;
  long long source_layer, source_seq, source_head;      // strides in elements; 0 where all layers, or all heads, share one list
  const int* count;
  float* weights;             // [layers][weight_slots][nkv][weight_width] or null: moved along
  long long weight_layer;
  int weight_width;
  int n_seqs, nkv, most;      // most: bound of count over the batch
};

#ifdef __CUDACC__
// Lets a kernel have `smem` bytes of dynamic shared memory, once per device: asked for at every launch it takes a third of a microsecond of a
// call that is bound by the host.  `done`: a static word of the caller's, one per kernel.
template <typename K>
static inline cudaError_t llg_allow_smem(K kernel, size_t smem, unsigned long long& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 63;
  if (dev < 63 && (__atomic_load_n(&done, __ATOMIC_RELAXED) >> dev & 1)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) __atomic_fetch_or(&done, 1ull << dev, __ATOMIC_RELAXED);
  return e;
}
#endif
