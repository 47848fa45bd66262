// What the two kernels of tree attention share: the sets of ancestors, the mask, the arguments.
#pragma once
#include "common.hpp"

namespace mi355 {

constexpr int TREE_MAX_NODES = 64;

struct TreeArgs {
  const half_t *q, *kc, *vc;
  const int *table, *seq_lens, *parents;
  half_t* out;
  float *part_acc, *part_ml;  // [S, N, Hq, splits, 128] and [.., 2]
  int num_kv_heads, group, nodes, max_pages, num_pages, page_shift, num_splits, chunk_steps;
  int ranked;  // walk the sequences longest first
  float scale_log2e;
};

// Ancestors (and self) of node `lane` as a bit set, by pointer doubling over one wave; a parent that does not come before
// its node is none.
__device__ __forceinline__ unsigned long long tree_ancestors(const int* parents, int nodes) {
  const int lane = threadIdx.x & 63;
  int up = lane < nodes ? parents[lane] : -1;
  up = (up >= 0 && up < lane) ? up : -1;
  unsigned long long set = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; i++) {
    const int from = up < 0 ? lane : up;
    const unsigned long long s = __shfl(set, from);
    const int next = __shfl(up, from);
    if (up >= 0) {
      set |= s;
      up = next;
    }
  }
  return set;
}

// Which of the four positions d, .. , d + 3 (counted from the first draft) a node with ancestor set `seen` sees, as bits 0 .. 3:
// all in front of the drafts, then the set's; the set has no bits behind the last draft.
__device__ __forceinline__ unsigned tree_visible4(unsigned long long seen, int d) {
  const int up = d > 0 ? (d < 63 ? d : 63) : 0, down = d < 0 ? (d > -4 ? -d : 4) : 0;
  const unsigned w = d > 63 ? 0u : (unsigned)(seen >> up);
  return (w << down) | ((1u << down) - 1u);
}

// v where bit r of `visible` is set, else -inf, by bit operations: the selection on a chain of conditions (dropped, behind
// the end, a draft that is no ancestor) has been compiled to one that keeps the score.
__device__ __forceinline__ float tree_hide(float v, unsigned visible, int r) {
  const unsigned keep = (unsigned)((int)(visible << (31 - r)) >> 31);
  return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, v) & keep) | (0xFF800000u & ~keep));
}

// The sequence of rank `rank` by falling length, at most 64 of them: one per lane, every wave by itself.
__device__ __forceinline__ int tree_rank(const int* seq_lens, int num_seqs, int rank) {
  const int lane = threadIdx.x & 63;
  const int len = lane < num_seqs ? seq_lens[lane] : 0;
  int before = 0;
  for (int j = 0; j < num_seqs; j++) {
    const int other = __builtin_amdgcn_readlane(len, j);
    before += other > len || (other == len && j < lane);
  }
  return __builtin_ctzll(__builtin_amdgcn_ballot_w64(before == rank && lane < num_seqs));
}

// The prefill kernel's tree form (flash_attn_fwd.hip): 64 or 128 query rows per workgroup.  chunk_steps even.
int fa_tree(const TreeArgs& a, int num_seqs, bool bf16, hipStream_t stream);

}  // namespace mi355
