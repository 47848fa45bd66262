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
  int num_kv_heads, group, nodes, max_pages, num_pages, page_shift, num_splits;
  int num_seqs;
  unsigned per_half;  // see tree_chunk_steps
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

// Bits 15 and 31 where the low and the high of two 16-bit numbers are infinite or NaN (an exponent of all ones).
template <bool BF>
__device__ __forceinline__ unsigned tree_nonfinite2(unsigned two) {
  return BF ? ((two & 0x7F807F80u) + 0x00800080u) & 0x80008000u : ((two & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
}

// The 16-bit number of these bits.
template <bool BF>
__device__ __forceinline__ float tree_value(unsigned bits) {
  return BF ? __builtin_bit_cast(float, bits << 16) : (float)__builtin_bit_cast(half_t, (unsigned short)bits);
}

// Chunks: 32-token steps in each, the same number in every workgroup and in the merge; even, and at least 128 tokens.  The longest
// sequence's steps over num_splits, not the block table's: a server's table is as wide as its longest context may get, and where
// its columns were cut (32 chunks of 131072) a sequence of 4096 tokens was one chunk on eight workgroups (56 us; 17 by its length).
// Above 512 sequences the table's width: a workgroup would look at lengths longer than that saves (1024 sequences of 100 tokens in
// two chunks 30.5 us by length, 22.4 by the table; 4096 of 600 499 and 234; the default is one chunk there).
constexpr int TREE_LENGTHS = 512;
__device__ __forceinline__ int tree_chunk_steps(const int* seq_lens, int num_seqs, int num_splits, unsigned per_half, int reach) {
  int longest = reach;
  if (num_splits > 1 && num_seqs <= TREE_LENGTHS) {
    int len = 0;
    if (num_seqs == 1) {
      len = seq_lens[0];
    } else {
      const int lane = threadIdx.x & 63;
      len = lane < num_seqs ? seq_lens[lane] : 0;  // (the load that tree_item needs too)
      if (num_seqs > 64) {  // all loads at once; lanes behind the last sequence take its length again
#pragma unroll
        for (int s = 64; s < TREE_LENGTHS; s += 64) {
          const int l = seq_lens[s + lane < num_seqs ? s + lane : num_seqs - 1];
          len = l > len ? l : len;
        }
      }
      auto with = [&](int l) { len = l > len ? l : len; };  // (lanes without a partner keep their own)
      with(__builtin_amdgcn_update_dpp(len, len, 0x111, 0xF, 0xF, false));  // row_shr:1, 2, 4, 8: lane 15 of each row has the row's
      with(__builtin_amdgcn_update_dpp(len, len, 0x112, 0xF, 0xF, false));
      with(__builtin_amdgcn_update_dpp(len, len, 0x114, 0xF, 0xF, false));
      with(__builtin_amdgcn_update_dpp(len, len, 0x118, 0xF, 0xF, false));
      with(__builtin_amdgcn_update_dpp(len, len, 0x142, 0xF, 0xF, false));  // row_bcast:15, 31: lane 63 has all
      with(__builtin_amdgcn_update_dpp(len, len, 0x143, 0xF, 0xF, false));
      len = __builtin_amdgcn_readlane(len, 63);
    }
    len = len > 0 ? len : 0;
    longest = len < reach ? len : reach;
  }
  // per_half = ceil(2^32 / (2 num_splits)): the quotient's whole part, or one more, which only makes chunks longer
  const int each = 2 * (int)__umulhi((unsigned)(((longest + 31) >> 5) + 2 * num_splits - 1), per_half);
  return each < 4 ? 4 : each;
}
inline unsigned tree_per_half(int64_t num_splits) { return (unsigned)(((1ll << 32) + 2 * num_splits - 1) / (2 * num_splits)); }

// Piece of work number `item` of a call whose sequences are cut into chunks of `chunk_steps` 32-token steps: its sequence and chunk;
// false behind the last.  Up to 64 sequences (one per lane, every wave by itself): all full chunks first, then the
// sequences' last chunks, the longest first, so that the short ones make up the tail.  Nothing empty lies between: workgroups
// go to a chip's shader engines in turn, full or not, and where every fourth one was an empty chunk (4 chunks a sequence,
// most of them shorter) three quarters of the chip did the work (255 against 182 us).  More sequences: chunk by chunk.
__device__ __forceinline__ bool tree_item(const int* seq_lens, int num_seqs, int num_splits, int chunk_steps, int reach, int item, int& seq, int& split) {
  if (num_seqs == 1 || num_seqs > 64) {
    split = item / num_seqs;
    seq = item - split * num_seqs;
    return split < num_splits;
  }
  const int lane = threadIdx.x & 63;
  int len = lane < num_seqs ? seq_lens[lane] : 0;
  len = len < 0 ? 0 : (len > reach ? reach : len);
  const int steps = (len + 31) >> 5;
  const int full = steps > 0 ? (steps - 1) / chunk_steps : 0;  // chunks in front of the last one
  const int last = lane < num_seqs ? steps - full * chunk_steps : -1;
  int before = 0, rank = 0, all = 0;
  for (int j = 0; j < num_seqs; j++) {
    const int fj = __builtin_amdgcn_readlane(full, j), lj = __builtin_amdgcn_readlane(last, j);
    before += j < lane ? fj : 0;
    all += fj;
    rank += lj > last || (lj == last && j < lane);
  }
  if (item >= all + num_seqs) return false;
  const bool mine = item < all ? (before <= item && item < before + full) : (rank == item - all && lane < num_seqs);
  seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine));
  split = item < all ? item - __builtin_amdgcn_readlane(before, seq) : __builtin_amdgcn_readlane(full, seq);
  return true;
}

// The prefill kernel's tree form (flash_attn_fwd.hip): 64 or 128 query rows per workgroup.
int fa_tree(const TreeArgs& a, int num_seqs, bool bf16, hipStream_t stream);

}  // namespace mi355
