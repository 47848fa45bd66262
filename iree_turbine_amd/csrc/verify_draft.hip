// Verification of drafted tokens against the target model's probabilities, from given random numbers.
//
// Per sequence the drafts form a tree (a chain is the tree whose nodes have one child each): node 0 is the last token
// that is certain, p_i the target's distribution behind node i, q_i the one node i's children were drawn from (a point
// mass on the child itself where no draft probabilities are given).  The walk starts at node 0 with r = p_0, M = 1 and
// tries the present node's children in index order:
//   accepted, where u_i M q(t_i) < r(t_i): the child is the present node, r = p_i, M = 1;
//   rejected otherwise:                     r <- max(r - M q, 0), M <- sum of r   (left as they are if that sum is 0).
// The next token is drawn from r behind the last try: the first v whose running sum of r exceeds u_0 times the total.
// Kept unnormalised, r after k rejections is max(p - A_k q, 0) with A_k = 1 + M_1 + ... + M_(k-1): one scalar.
//
// All of it is computed in 64 bits: products of two 32-bit numbers are exact there, and a sum over the vocabulary is
// good to 1e-16, so the outcome does not hang on the order of a sum.
//
// A walk needs single elements of p and q up to its first rejection (or its end), then sums over rows of the
// vocabulary.  HBM bound where many sequences end in one row each, latency bound otherwise.  Two launches:
//   sums: chunks of the vocabulary x sequences; every workgroup repeats the walk to its first stop (two dependent
//         loads and N steps in registers) and sums its chunk of the row it stopped at;
//   walk: one workgroup per sequence; continues from those sums, makes further passes itself where siblings are
//         rejected one after the other, and finds the token inside the one chunk that holds it.
#include "common.hpp"
#include <math.h>

namespace mi355 {

constexpr int VD_CHUNK = 4096;      // vocabulary entries per partial sum
constexpr int VD_SUM_THREADS = 256;
constexpr int VD_WALK_THREADS = 1024;
constexpr int VD_MAX_NODES = 64;    // one lane per node

struct VdArgs {
  const float* target;   // [S, N, V]
  const float* draft;    // [S, N, V] or null: point masses
  const int* tokens;     // [S, N]
  const int* parents;    // [S, N]
  const float* uniforms; // [S, N]
  int N, V, chunks;
};

// What the walk knows, the same in every lane but for the first six members (lane i: node i).
struct VdWalk {
  int parent, token;
  double u, p, q, r;      // p, q at the node's token in its parent's rows; r: the residual there
  int cur, count, next;   // present node, accepted so far, next node to try
  int path;               // lane k: the k-th accepted node
  int rejected;           // rejections that changed r at the present node
  double mass, all;       // M and A
};

__device__ __forceinline__ double vd_lane(double v, int lane) {
  return __shfl(v, lane);
}

__device__ __forceinline__ VdWalk vd_begin(const VdArgs& a, long long seq) {
  VdWalk w;
  const int lane = threadIdx.x & 63;
  const bool on = lane < a.N;
  const long long base = seq * a.N;
  w.parent = (on && lane > 0) ? a.parents[base + lane] : -1;
  w.token = on ? a.tokens[base + lane] : 0;
  w.u = on ? (double)a.uniforms[base + lane] : 0.0;
  // a node whose parent does not come before it, or whose token is none, is nobody's child
  if (w.parent < 0 || w.parent >= lane || w.token < 0 || w.token >= a.V) w.parent = -1;
  w.p = w.q = 0.0;
  if (w.parent >= 0) {
    const long long at = (base + w.parent) * a.V + w.token;
    w.p = (double)a.target[at];
    w.q = a.draft ? (double)a.draft[at] : 1.0;
  }
  w.r = w.p;
  w.cur = 0, w.count = 0, w.next = 1, w.path = -1;
  w.rejected = 0, w.mass = 1.0, w.all = 0.0;
  return w;
}

// Tries nodes until one is rejected (returns it) or none is left (returns -1).
__device__ __forceinline__ int vd_advance(const VdArgs& a, VdWalk& w) {
  const int lane = threadIdx.x & 63;
  while (w.next < a.N) {
    const unsigned long long children = __builtin_amdgcn_ballot_w64(w.parent == w.cur && lane >= w.next);
    if (children == 0) {
      w.next = a.N;
      break;
    }
    const int i = __builtin_ctzll(children);
    w.next = i + 1;
    const double u = vd_lane(w.u, i), q = vd_lane(w.q, i), r = vd_lane(w.r, i);
    if (!(u * (q * w.mass) < r)) return i;
    if (lane == w.count) w.path = i;
    w.count++;
    w.cur = i;
    w.rejected = 0, w.mass = 1.0, w.all = 0.0;
  }
  return -1;
}

// The rejection of node i left `total` > 0.
__device__ __forceinline__ void vd_reject(const VdArgs& a, VdWalk& w, int i, double total) {
  if (a.draft) {
    if (w.parent == w.cur) w.r = fmax(w.p - (w.all + w.mass) * w.q, 0.0);
  } else {
    const int tok = __shfl(w.token, i);
    if (w.parent == w.cur && w.token == tok) w.r = fmax(w.r - w.mass, 0.0);
  }
  w.rejected++;
  w.all += w.mass;
  w.mass = total;
}

// The residual at entry v of the present node's rows, after `n` rejections of which the first n have factor A = all
// (drafts with probabilities) or the tokens tok[0 .. n) and what they took away (point masses).
struct VdResid {
  const float *p, *q;
  double all;
  int n;
  const int* tok;
  const double* sub;
  __device__ __forceinline__ double at(int v) const {
    double r = (double)p[v];
    if (n == 0) return r;
    if (q) return fmax(r - all * (double)q[v], 0.0);
    for (int k = 0; k < n; k++)
      if (tok[k] == v) r = fmax(r - sub[k], 0.0);
    return r;
  }
};

// Sum over the workgroup, the same value in every thread; a fixed order.
template <int WAVES>
__device__ __forceinline__ double vd_block_sum(double v, double* tmp) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) s += tmp[w];
  __syncthreads();
  return s;
}

__global__ __launch_bounds__(VD_SUM_THREADS) void verify_sums_kernel(VdArgs a, double* __restrict__ sums) {
  __shared__ double tmp[VD_SUM_THREADS / 64], sub[1];
  __shared__ int tok[1];
  const long long seq = blockIdx.y;
  VdWalk w = vd_begin(a, seq);
  const int i = vd_advance(a, w);
  const long long row = (seq * a.N + w.cur) * a.V;
  VdResid res{a.target + row, a.draft ? a.draft + row : nullptr, 0.0, 0, tok, sub};
  if (i >= 0) {
    res.n = 1, res.all = 1.0;
    if (!a.draft) {
      const int t = __shfl(w.token, i);
      if (threadIdx.x == 0) tok[0] = t, sub[0] = 1.0;
      __syncthreads();
    }
  }
  const int v0 = blockIdx.x * VD_CHUNK;
  const int v1 = a.V - v0 > VD_CHUNK ? v0 + VD_CHUNK : a.V;
  double s = 0.0;
  for (int v = v0 + (int)threadIdx.x; v < v1; v += VD_SUM_THREADS) s += res.at(v);
  s = vd_block_sum<VD_SUM_THREADS / 64>(s, tmp);
  if (threadIdx.x == 0) sums[seq * a.chunks + blockIdx.x] = s;
}

__global__ __launch_bounds__(VD_WALK_THREADS) void verify_walk_kernel(VdArgs a, double* __restrict__ sums, int* __restrict__ path,
                                                                      int* __restrict__ accepted, int* __restrict__ next_token) {
  constexpr int WAVES = VD_WALK_THREADS / 64;
  __shared__ double tmp[WAVES], sub[VD_MAX_NODES];
  __shared__ int tok[VD_MAX_NODES], found[2];
  const long long seq = blockIdx.x;
  const int t = threadIdx.x, lane = t & 63;
  double* part = sums + seq * a.chunks;

  // chunk sums of a residual into `part`, and their total
  auto total_of = [&]() {
    double s = 0.0;
    for (int c = t; c < a.chunks; c += VD_WALK_THREADS) s += part[c];
    return vd_block_sum<WAVES>(s, tmp);
  };
  auto make_sums = [&](const VdResid& res) {
    __syncthreads();
    for (int c = t >> 6; c < a.chunks; c += WAVES) {
      const int v0 = c * VD_CHUNK, v1 = a.V - v0 > VD_CHUNK ? v0 + VD_CHUNK : a.V;
      double s = 0.0;
      for (int v = v0 + lane; v < v1; v += 64) s += res.at(v);
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
      if (lane == 0) part[c] = s;
    }
    __syncthreads();
    return total_of();
  };
  VdWalk w = vd_begin(a, seq);
  auto resid = [&](int n, double all) {
    const long long row = (seq * a.N + w.cur) * a.V;
    return VdResid{a.target + row, a.draft ? a.draft + row : nullptr, all, n, tok, sub};
  };

  bool given = true;   // `part` holds the sums that the first stop of the walk asks for
  bool ready = false;  // `part` holds the sums of r, `total` their total
  double total = 0.0;
  for (;;) {
    const int i = vd_advance(a, w);
    if (i < 0) break;
    if (!a.draft) {
      const int rejected_tok = __shfl(w.token, i);
      if (t == 0) tok[w.rejected] = rejected_tok, sub[w.rejected] = w.mass;
      __syncthreads();
    }
    const double left = given ? total_of() : make_sums(resid(w.rejected + 1, w.all + w.mass));
    given = false;
    ready = left > 0.0;
    if (ready) {
      vd_reject(a, w, i, left);
      total = left;
    }
  }
  // accepted nodes since the last sums, or a rejection that left nothing: the sums are those of another residual
  if (w.rejected == 0) ready = false;
  if (!ready) total = given ? total_of() : make_sums(resid(w.rejected, w.all));

  if (t < 64 && t < a.N) path[seq * a.N + t] = w.path;
  if (t == 0) accepted[seq] = w.count;

  // the chunk that holds the token, then the token
  const double u0 = vd_lane(w.u, 0);
  const double goal = (u0 > 0.0 ? u0 : 0.0) * total;
  int token = -1;
  if (total > 0.0) {
    if (t == 0) {
      double run = 0.0;
      int c = -1, last = 0;
      double before = 0.0, before_last = 0.0;
      for (int k = 0; k < a.chunks; k++) {
        const double s = part[k];
        if (s > 0.0) last = k, before_last = run;
        run += s;
        if (run > goal) {
          c = k, before = run - s;
          break;
        }
      }
      if (c < 0) c = last, before = before_last;
      found[0] = c;
      tmp[0] = before;
    }
    __syncthreads();
    const int c = found[0];
    const double before = tmp[0];
    __syncthreads();
    const VdResid res = resid(w.rejected, w.all);
    const int v0 = c * VD_CHUNK, v1 = a.V - v0 > VD_CHUNK ? v0 + VD_CHUNK : a.V;
    if (t == 0) found[0] = 0x7fffffff, found[1] = -1;
    // VD_CHUNK / VD_WALK_THREADS neighbours per thread
    constexpr int PER = VD_CHUNK / VD_WALK_THREADS;
    double r[PER], mine = 0.0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int v = v0 + t * PER + k;
      r[k] = v < v1 ? res.at(v) : 0.0;
      mine += r[k];
    }
    double incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    if (lane == 63) tmp[t >> 6] = incl;
    __syncthreads();
    double run = before;
#pragma unroll
    for (int x = 0; x < WAVES; x++) run += x < (t >> 6) ? tmp[x] : 0.0;
    run += incl - mine;
    int hit = 0x7fffffff, any = -1;
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int v = v0 + t * PER + k;
      run += r[k];
      if (r[k] > 0.0) {
        any = v;
        if (run > goal && v < hit) hit = v;
      }
    }
    if (hit != 0x7fffffff) atomicMin(&found[0], hit);
    if (any >= 0) atomicMax(&found[1], any);
    __syncthreads();
    // rounding may leave none in the chunk: its last entry with mass
    token = found[0] != 0x7fffffff ? found[0] : found[1];
  }
  if (t == 0) next_token[seq] = token;
}

}  // namespace mi355

using namespace mi355;

static int64_t vd_chunks(int64_t V) { return (V + VD_CHUNK - 1) / VD_CHUNK; }

static bool vd_sizes_ok(int64_t S, int64_t N, int64_t V) {
  return S > 0 && S <= 65535 && N > 0 && N <= VD_MAX_NODES && V > 0 && V <= (1 << 24);
}

extern "C" int64_t mi355_verify_draft_workspace_bytes(int64_t num_seqs, int64_t num_nodes, int64_t vocab) {
  if (!vd_sizes_ok(num_seqs, num_nodes, vocab)) return 0;
  return num_seqs * vd_chunks(vocab) * (int64_t)sizeof(double);
}

extern "C" int mi355_verify_draft(const float* target_probs, const float* draft_probs, const int32_t* tokens, const int32_t* parents,
                                  const float* uniforms, int32_t* path, int32_t* num_accepted, int32_t* next_token,
                                  int64_t num_seqs, int64_t num_nodes, int64_t vocab, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  const char* fn = "verify_draft";
  if (!target_probs || !tokens || !parents || !uniforms || !path || !num_accepted || !next_token)
    return fail(-MI355_E_NULL, "%s: null pointer", fn);
  if (!vd_sizes_ok(num_seqs, num_nodes, vocab))
    return fail(-MI355_E_SHAPE, "%s: bad sizes seqs=%lld nodes=%lld (1 to %d) vocab=%lld", fn, (long long)num_seqs, (long long)num_nodes,
                VD_MAX_NODES, (long long)vocab);
  if (!workspace || workspace_bytes < mi355_verify_draft_workspace_bytes(num_seqs, num_nodes, vocab))
    return fail(-MI355_E_SCRATCH, "%s: workspace missing or too small", fn);
  if (!aligned16(workspace)) return fail(-MI355_E_ALIGN, "%s: workspace must be 16-byte aligned", fn);
  const VdArgs a{target_probs, draft_probs, tokens, parents, uniforms, (int)num_nodes, (int)vocab, (int)vd_chunks(vocab)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  dim3 grid((unsigned)a.chunks, (unsigned)num_seqs), block(VD_SUM_THREADS);
  hipLaunchKernelGGL(verify_sums_kernel, grid, block, 0, s, a, (double*)workspace);
  if (int rc = check_launch("verify_sums_kernel", grid, block, 0)) return rc;
  dim3 grid2((unsigned)num_seqs), block2(VD_WALK_THREADS);
  hipLaunchKernelGGL(verify_walk_kernel, grid2, block2, 0, s, a, (double*)workspace, path, num_accepted, next_token);
  return check_launch("verify_walk_kernel", grid2, block2, 0);
}
