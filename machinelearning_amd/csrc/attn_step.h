// A cached attention step whose sequences have lengths of their own, whose active block
// may be a tree, and whose heads may hold two softmax maps (attn_diff.h): parameters and
// the pieces that its kernels share.
//
// Sequence b's keys are the first Lc = lens[b] rows of its cache and then the block's T
// rows. Every query in the tree sees the Lc rows; of the block, query t sees its line of
// descent (itself, its parent, ...) where `parents` is given, and keys <= t (causal) or
// all T otherwise. Keys are walked in blocks of 32: ceil(Lc / 32) of the cache, then
// ceil(T / 32) of the block, so that word w of a query's visibility is block w's mask.
#pragma once

#include "attn_common.h"

namespace mi {

struct StepParams {
  int B, T, H, Hkv, rep;
  int rows;                            // rows that a sequence's cache can hold
  int causal;                          // without parents: 1 chain, 0 every key of the block
  float scale, scale_log2;
  long long k_sb, k_sh, v_sb, v_sh;    // cache strides (elements); rows are D apart
  const int* lens;                     // [B] cached rows (nullptr: `rows` each)
  const int* parents;                  // [B, T] (nullptr: no tree)
  int parents_sb;                      // T, or 0: one tree for every sequence
  const float* gate;                   // [B, T, H] output gate logits (nullptr: none)
  const void* lam;                     // [H] map weights (two maps only)
  int lam_dtype;
  int R;                               // query rows per kv head: T * rep
  int nsplit;                          // workgroups
  bool direct;                         // a workgroup per unit
  int min_blocks;                      // key blocks that a workgroup takes at least
  float resc_th;                       // lazy-rescale threshold in raw score units
  FastDiv div_rep, div_ups, div_ngrp;  // by rep, units per sequence, row groups
};

constexpr int kTreeMax = 256;          // nodes of a tree: one per thread of a workgroup
constexpr int kTreeWords = kTreeMax / 32;
constexpr float kStepNegInit = -1e30f; // finite running-max sentinel

// Lines of descent of a tree, in LDS.
struct TreeLds {
  unsigned line[kTreeMax][kTreeWords + 1];   // bit a of node t: t sees node a (padded rows)
  int up[kTreeMax];                          // after build: -1 in the tree, -2 not
};

// Fills `s` by pointer doubling: after i rounds a node's line holds its 2^i nearest
// ancestors and `up` the one after them, so a line of any depth takes log2 T rounds. A
// parent other than -1 that is not an earlier node puts a node, and with it every node
// under it, outside the tree (up = -2): such nodes see nothing and nobody sees them.
// All threads of a workgroup of at least kTreeMax.
__device__ __forceinline__ void tree_build(TreeLds& s, const StepParams& p, int b) {
  const int t = threadIdx.x, W = (p.T + 31) / 32;
  const bool node = t < p.T;
  unsigned w[kTreeWords];
  int up = -2;
  if (node) {
    const int x = p.parents[(long long)b * p.parents_sb + t];
    up = x >= -1 && x < t ? x : -2;
#pragma unroll
    for (int i = 0; i < kTreeWords; ++i) {
      w[i] = i == t / 32 ? 1u << (t & 31) : 0u;
      if (i < W) s.line[t][i] = w[i];
    }
    s.up[t] = up;
  }
  __syncthreads();
  while (true) {
    const bool more = node && up >= 0;
    if (!__syncthreads_or(more)) break;
    int next = up;
    if (more) {
#pragma unroll
      for (int i = 0; i < kTreeWords; ++i)
        if (i < W) w[i] |= s.line[up][i];
      next = s.up[up];
    }
    __syncthreads();
    if (more) {
      up = next;
#pragma unroll
      for (int i = 0; i < kTreeWords; ++i)
        if (i < W) s.line[t][i] = w[i];
      s.up[t] = up;
    }
    __syncthreads();
  }
}

// Block `w`'s keys of the active block that query t sees, without a tree.
__device__ __forceinline__ unsigned chain_word(const StepParams& p, int t, int w) {
  const int last = (p.causal ? min(t, p.T - 1) : p.T - 1) - 32 * w;
  return last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
}

__device__ __forceinline__ int step_len(const StepParams& p, int b) {
  return p.lens ? min(max(p.lens[b], 0), p.rows) : p.rows;
}

}  // namespace mi
