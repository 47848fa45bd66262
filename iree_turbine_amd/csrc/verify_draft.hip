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
// vocabulary, one row after the other.  HBM bound where many sequences end in one row each, latency bound otherwise.
//   sums (one launch, or up to four): pieces of the vocabulary x sequences; every workgroup repeats the walk up to the sum
//         that is wanted next (two dependent loads and a few steps in registers; totals of earlier launches are added up
//         from their pieces) and sums its pieces of that row; a sequence that wants no more says so in a word that the
//         next launch looks at first;
//   walk: one workgroup per sequence; the same walk to its end, from those sums as far as they go, then with passes of its own,
//         and the token: a scan over the last row's pieces, and one wave inside the piece.
// A pass by the one workgroup is bound by its CU's rate of 64-bit operations (131072 entries: 25 us, about 100 cycles per 64
// entries), a launch of sums by memory (13 us for 64 sequences) and costs 3 us where no sequence needs it: calls that can
// reject a second sibling and have 65536 entries or more get up to four launches of sums, others one.
// A row's sums are kept per piece of 256 entries (more above 2^18 entries, so that there are at most 1024): 64 lanes of 16
// bytes, four pieces at a time and the next four requested ahead (4-byte loads one at a time: 75 us a pass).
#include "common.hpp"
#include <math.h>

namespace mi355 {

constexpr int VD_BLOCK = 256;        // vocabulary entries that one wave takes at a time
constexpr int VD_MAX_PIECES = 1024;  // sums per row
constexpr int VD_GROUP = 128;        // sums that one wave adds up, two per lane
constexpr int VD_AHEAD = 4;          // pieces that a wave has in flight
constexpr int VD_SUM_THREADS = 256;
constexpr int VD_SUM_PIECES = VD_SUM_THREADS / 64 * VD_AHEAD;  // pieces that a workgroup of a launch of sums has in flight
constexpr int VD_WALK_THREADS = VD_MAX_PIECES / 2;
constexpr int VD_MAX_NODES = 64;     // one lane per node

struct VdArgs {
  const float* target;   // [S, N, V]
  const float* draft;    // [S, N, V] or null: point masses
  const int* tokens;     // [S, N]
  const int* parents;    // [S, N]
  const float* uniforms; // [S, N]
  int N, V, pieces, blocks;  // a piece is `blocks` blocks; blocks == 1 up to 2^18 entries
};

// What the walk knows, the same in every lane but for the first seven members (lane i: node i).
struct VdWalk {
  int parent, token;
  double u, p, q, r;       // p, q at the node's token in its parent's rows; r: the residual there
  int path;                // lane k: the k-th accepted node
  int cur, count, next;    // present node, accepted so far, next node to try
  int tried;               // the node whose rejection waits for a sum, -1: the walk is at its end
  int rejected;            // rejections that changed r at the present node
  bool ready;              // the last sums asked for are those of r
  double mass, all;        // M and A
};

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
  w.cur = 0, w.count = 0, w.next = 1, w.tried = -1, w.path = -1;
  w.rejected = 0, w.ready = false, w.mass = 1.0, w.all = 0.0;
  return w;
}

// Goes on to the next row sum that the walk needs: of the residual that the rejection of w.tried would leave, or at the end
// (w.tried < 0) of r; false if the last sums asked for are those of r already.
__device__ __forceinline__ bool vd_ask(const VdArgs& a, VdWalk& w) {
  const int lane = threadIdx.x & 63;
  w.tried = -1;
  for (;;) {
    const unsigned long long left = w.next < a.N ? ~0ull << w.next : 0ull;
    const unsigned long long children = __builtin_amdgcn_ballot_w64(w.parent == w.cur) & left;
    if (children == 0) break;
    const int i = __builtin_ctzll(children);
    w.next = i + 1;
    if (!((__builtin_amdgcn_ballot_w64(w.u * (w.q * w.mass) < w.r) >> i) & 1)) {
      w.tried = i;
      return true;
    }
    if (lane == w.count) w.path = i;
    w.count++;
    w.cur = i;
    w.rejected = 0, w.ready = false, w.mass = 1.0, w.all = 0.0;
  }
  return !w.ready;
}

// The sum that was asked for; false when the walk is over.
__device__ __forceinline__ bool vd_answer(const VdArgs& a, VdWalk& w, double total) {
  if (w.tried < 0) return false;
  w.ready = total > 0.0;
  if (w.ready) {
    if (a.draft) {
      if (w.parent == w.cur) w.r = fmax(__builtin_fma(-(w.all + w.mass), w.q, w.p), 0.0);
    } else {
      const int tok = __builtin_amdgcn_readlane(w.token, w.tried);
      if (w.parent == w.cur && w.token == tok) w.r = fmax(w.r - w.mass, 0.0);
    }
    w.rejected++;
    w.all += w.mass;
    w.mass = total;
  }
  return true;
}

// The residual of the present node's rows after `n` rejections: p (none), p - A q (drafts with probabilities), or p less
// what the tokens tok[0 .. n) had (point masses).  The kind is chosen outside the loops over a row.
enum class VdKind { PLAIN, FACTOR, POINTS };
struct VdResid {
  const float *p, *q;
  double all;
  int n;
  const int* tok;
  const double* sub;
  __device__ __forceinline__ VdKind kind() const { return n == 0 ? VdKind::PLAIN : q ? VdKind::FACTOR : VdKind::POINTS; }
  template <VdKind K>
  __device__ __forceinline__ double of(float pv, float qv, int v) const {
    double r = (double)pv;
    if constexpr (K == VdKind::FACTOR) r = fmax(__builtin_fma(-all, (double)qv, r), 0.0);
    if constexpr (K == VdKind::POINTS)
      for (int k = 0; k < n; k++)
        if (tok[k] == v) r = fmax(r - sub[k], 0.0);
    return r;
  }
};

// Four neighbouring entries of a row; rows lie on 4-byte borders only.
struct alignas(4) VdFour { float v[4]; };

// The four entries from v on of both rows (zeros behind the row's end, at V).
template <VdKind K>
__device__ __forceinline__ void vd_load4(const VdResid& res, int v, int V, VdFour& p, VdFour& q) {
  if (v + 4 <= V) {
    p = *reinterpret_cast<const VdFour*>(res.p + v);
    if constexpr (K == VdKind::FACTOR) q = *reinterpret_cast<const VdFour*>(res.q + v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      p.v[e] = v + e < V ? res.p[v + e] : 0.f;
      if constexpr (K == VdKind::FACTOR) q.v[e] = v + e < V ? res.q[v + e] : 0.f;
    }
  }
}

// One step of a wave: VD_AHEAD pieces' next blocks.
template <VdKind K>
struct VdBatch {
  VdFour p[VD_AHEAD], q[VD_AHEAD];
  __device__ __forceinline__ void load(const VdArgs& a, const VdResid& res, int first, int step, int b) {
#pragma unroll
    for (int k = 0; k < VD_AHEAD; k++) {
      const int piece = first + k * step;
      p[k] = VdFour{}, q[k] = VdFour{};
      if (piece < a.pieces) vd_load4<K>(res, (piece * a.blocks + b) * VD_BLOCK + (threadIdx.x & 63) * 4, a.V, p[k], q[k]);
    }
  }
};

// Sums of the residual over the pieces first, first + step, .. below a.pieces, handed to put(piece, sum) in one lane each.
// The next batch is requested before the present one is added up.
template <VdKind K, typename F>
__device__ __forceinline__ void vd_piece_sums(const VdArgs& a, const VdResid& res, int first, int step, F&& put) {
  static_assert(VD_AHEAD == 4, "the sums of a batch are added up by four groups of lanes");
  const int lane = threadIdx.x & 63;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  VdBatch<K> now, next;
  int b = 0;
  now.load(a, res, first, step, 0);
  while (first < a.pieces) {
    int first_next = first, b_next = b + 1;
    if (b_next == a.blocks) first_next += 4 * step, b_next = 0;
    if (first_next < a.pieces) next.load(a, res, first_next, step, b_next);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int v = ((first + k * step) * a.blocks + b) * VD_BLOCK + lane * 4;
#pragma unroll
      for (int e = 0; e < 4; e++) s[k] += res.of<K>(now.p[k].v[e], now.q[k].v[e], v + e);
    }
    if (b_next == 0) {
      // sixteen lanes end up with each sum: 7 exchanges instead of 24
      const bool h5 = lane & 32, h4 = lane & 16;
      double x = h5 ? s[2] : s[0], y = h5 ? s[3] : s[1];
      x += __shfl_xor(h5 ? s[0] : s[2], 32);
      y += __shfl_xor(h5 ? s[1] : s[3], 32);
      double z = h4 ? y : x;
      z += __shfl_xor(h4 ? x : y, 16);
#pragma unroll
      for (int d = 8; d >= 1; d >>= 1) z += __shfl_xor(z, d);
      const int piece = first + (lane >> 4) * step;
      if ((lane & 15) == 0 && piece < a.pieces) put(piece, z);
#pragma unroll
      for (int k = 0; k < 4; k++) s[k] = 0.0;
    }
    now = next;
    first = first_next, b = b_next;
  }
}
template <typename F>
__device__ __forceinline__ void vd_row_sums(const VdArgs& a, const VdResid& res, int first, int step, F&& put) {
  const VdKind kind = res.kind();
  if (kind == VdKind::PLAIN) vd_piece_sums<VdKind::PLAIN>(a, res, first, step, put);
  else if (kind == VdKind::FACTOR) vd_piece_sums<VdKind::FACTOR>(a, res, first, step, put);
  else vd_piece_sums<VdKind::POINTS>(a, res, first, step, put);
}

// The first entry of a piece at which the running sum, from `run` on, exceeds the goal, by one wave; if rounding leaves
// none, its last entry with mass.
template <VdKind K>
__device__ __forceinline__ int vd_find(const VdArgs& a, const VdResid& res, int piece, double run, double goal) {
  const int lane = threadIdx.x & 63;
  int hit = 0x7fffffff, any = -1;
  for (int b = 0; b < a.blocks && hit == 0x7fffffff; b++) {
    const int v = (piece * a.blocks + b) * VD_BLOCK + lane * 4;
    VdFour p = {}, q = {};
    vd_load4<K>(res, v, a.V, p, q);
    double r[4], four = 0.0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      r[e] = res.of<K>(p.v[e], q.v[e], v + e);
      four += r[e];
    }
    double upto = four;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double up = __shfl_up(upto, d);
      if (lane >= d) upto += up;
    }
    double here = run + (upto - four);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      here += r[e];
      if (r[e] > 0.0) {
        any = v + e;
        if (here > goal && hit == 0x7fffffff) hit = v + e;
      }
    }
    run += __shfl(upto, 63);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const int h = __shfl_xor(hit, d), n = __shfl_xor(any, d);
      hit = h < hit ? h : hit;
      any = n > any ? n : any;
    }
  }
  return hit != 0x7fffffff ? hit : any;
}

// The rows that vd_ask asked for.  Point masses: the rejected tokens and what they had go into tok and sub, which the
// workgroup shares.
__device__ __forceinline__ VdResid vd_asked(const VdArgs& a, const VdWalk& w, long long seq, int* tok, double* sub) {
  const long long row = (seq * a.N + w.cur) * a.V;
  const bool more = w.tried >= 0;
  if (!a.draft && more) {
    const int t = __builtin_amdgcn_readlane(w.token, w.tried);
    if (threadIdx.x == 0) tok[w.rejected] = t, sub[w.rejected] = w.mass;
    __syncthreads();
  }
  return VdResid{a.target + row, a.draft ? a.draft + row : nullptr, more ? w.all + w.mass : w.all, w.rejected + more, tok, sub};
}

// Total of a row's sums, the same bits in every thread of either kernel: groups of VD_GROUP in order, two sums per lane.
// `of(group)` gives a lane's two; tmp holds VD_MAX_PIECES / VD_GROUP values.
template <int THREADS, typename F>
__device__ __forceinline__ double vd_total(double* tmp, F&& of) {
  constexpr int GROUPS = VD_MAX_PIECES / VD_GROUP;
  for (int g = threadIdx.x >> 6; g < GROUPS; g += THREADS / 64) {
    const double2 two = of(g);
    double s = two.x + two.y;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) tmp[g] = s;
  }
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int g = 0; g < GROUPS; g++) s += tmp[g];
  __syncthreads();
  return s;
}
__device__ __forceinline__ double2 vd_two(const double* sums, int pieces, int first) {
  return double2{first < pieces ? sums[first] : 0.0, first + 1 < pieces ? sums[first + 1] : 0.0};
}

// Launch number `round` of the sums, [rounds][S][pieces].  stop[s]: so many of them sequence s has (or will need), as far as
// known; a launch reads what the ones before it wrote, and what its own workgroups write changes nothing for the others.
__global__ __launch_bounds__(VD_SUM_THREADS) void verify_sums_kernel(VdArgs a, double* __restrict__ sums, int* __restrict__ stop,
                                                                     int round, int batches) {
  __shared__ double tmp[VD_MAX_PIECES / VD_GROUP], sub[VD_MAX_NODES];
  __shared__ int tok[VD_MAX_NODES];
  const long long seq = blockIdx.y, num_seqs = gridDim.y;
  const int lane = threadIdx.x & 63;
  if (round > 0 && stop[seq] <= round) return;
  const bool lead = blockIdx.x == 0 && threadIdx.x == 0;
  VdWalk w = vd_begin(a, seq);
  bool more = vd_ask(a, w);  // always true: a walk asks at least once
  for (int k = 0; k < round; k++) {
    vd_asked(a, w, seq, tok, sub);
    const double* done = sums + (k * num_seqs + seq) * a.pieces;
    more = vd_answer(a, w, vd_total<VD_SUM_THREADS>(tmp, [&](int g) { return vd_two(done, a.pieces, g * VD_GROUP + 2 * lane); })) && vd_ask(a, w);
    if (!more) {
      if (lead) stop[seq] = k + 1;
      return;
    }
  }
  const VdResid res = vd_asked(a, w, seq, tok, sub);
  // the last one: the walk's end, or the rejection of a last child (unless it leaves nothing; the walk sees to that)
  const bool last = w.tried < 0 || (w.next < a.N ? __builtin_amdgcn_ballot_w64(w.parent == w.cur) >> w.next : 0) == 0;
  if (lead) stop[seq] = last ? round + 1 : 0x7fffffff;
  // a workgroup's pieces lie next to each other, a wave's in `batches` batches
  VdArgs mine = a;
  const int per_wave = VD_AHEAD * batches;
  const int first = (blockIdx.x * (VD_SUM_THREADS / 64) + (threadIdx.x >> 6)) * per_wave;
  mine.pieces = a.pieces < first + per_wave ? a.pieces : first + per_wave;
  double* out = sums + (round * num_seqs + seq) * a.pieces;
  if (first < a.pieces) vd_row_sums(mine, res, first, 1, [&](int piece, double s) { out[piece] = s; });
}

__global__ __launch_bounds__(VD_WALK_THREADS) void verify_walk_kernel(VdArgs a, const double* __restrict__ sums,
                                                                      const int* __restrict__ stop, int rounds,
                                                                      int* __restrict__ path, int* __restrict__ accepted,
                                                                      int* __restrict__ next_token) {
  constexpr int WAVES = VD_WALK_THREADS / 64;
  __shared__ double part[VD_MAX_PIECES], tmp[WAVES], sub[VD_MAX_NODES];
  __shared__ int tok[VD_MAX_NODES], found[2];
  const long long seq = blockIdx.x, num_seqs = gridDim.x;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;

  // thread t holds the sums of pieces 2 t and 2 t + 1
  double2 mine = vd_two(sums + seq * a.pieces, a.pieces, 2 * t);
  if (rounds > 1) rounds = stop[seq] < rounds ? stop[seq] : rounds;
  VdWalk w = vd_begin(a, seq);
  VdResid res{};
  double total = 0.0;
  for (int k = 0; vd_ask(a, w); k++) {
    res = vd_asked(a, w, seq, tok, sub);
    if (k >= rounds) {
      vd_row_sums(a, res, wave, WAVES, [&](int piece, double s) { part[piece] = s; });
      __syncthreads();
      mine = vd_two(part, a.pieces, 2 * t);
    } else if (k > 0) {
      mine = vd_two(sums + (k * num_seqs + seq) * a.pieces, a.pieces, 2 * t);
    }
    total = vd_total<VD_WALK_THREADS>(tmp, [&](int) { return mine; });
    if (!vd_answer(a, w, total)) break;
  }
  // res, mine and total are r's now
  if (t < 64 && t < a.N) path[seq * a.N + t] = w.path;
  if (t == 0) accepted[seq] = w.count;

  // the piece that holds the token: the first whose running sum exceeds the goal, or the last one with mass
  const unsigned long long u_bits = __builtin_bit_cast(unsigned long long, w.u);
  const double u0 = __builtin_bit_cast(double, (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)u_bits) |
                                                   (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(u_bits >> 32)) << 32);
  const double goal = (u0 > 0.0 ? u0 : 0.0) * total;
  double incl = mine.x + mine.y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 63) tmp[wave] = incl;
  if (t == 0) found[0] = 0x7fffffff, found[1] = -1;
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int x = 0; x < WAVES; x++) before += x < wave ? tmp[x] : 0.0;
  before += incl - (mine.x + mine.y);
  if (mine.x > 0.0 || mine.y > 0.0) {
    const bool in0 = mine.x > 0.0 && before + mine.x > goal, in1 = mine.y > 0.0 && before + mine.x + mine.y > goal;
    if (in0 || in1) atomicMin(&found[0], in0 ? 2 * t : 2 * t + 1);
    atomicMax(&found[1], mine.y > 0.0 ? 2 * t + 1 : 2 * t);
  }
  __syncthreads();
  const int piece = found[0] != 0x7fffffff ? found[0] : found[1];
  if (piece < 0 || !(total > 0.0)) {  // no mass (or not a number)
    if (t == 0) next_token[seq] = -1;
    return;
  }
  if (t == piece / 2) tmp[0] = piece & 1 ? before + mine.x : before;
  __syncthreads();
  if (wave != 0) return;
  const VdKind kind = res.kind();
  const double run = tmp[0];
  const int token = kind == VdKind::PLAIN    ? vd_find<VdKind::PLAIN>(a, res, piece, run, goal)
                    : kind == VdKind::FACTOR ? vd_find<VdKind::FACTOR>(a, res, piece, run, goal)
                                             : vd_find<VdKind::POINTS>(a, res, piece, run, goal);
  if (lane == 0) next_token[seq] = token;
}

}  // namespace mi355

using namespace mi355;

static int64_t vd_blocks(int64_t V) { return (V + (int64_t)VD_BLOCK * VD_MAX_PIECES - 1) / ((int64_t)VD_BLOCK * VD_MAX_PIECES); }
static int64_t vd_pieces(int64_t V) { return (V + vd_blocks(V) * VD_BLOCK - 1) / (vd_blocks(V) * VD_BLOCK); }

// launches of sums: of N - 1 tries each can want one.  From 65536 entries on a pass by a workgroup costs more than a launch
// that nobody needs.
static int vd_rounds(int64_t N, int64_t V) { return V < 65536 || N <= 2 ? 1 : N - 1 < 4 ? (int)N - 1 : 4; }

static bool vd_sizes_ok(int64_t S, int64_t N, int64_t V) {
  return S > 0 && S <= 65535 && N > 0 && N <= VD_MAX_NODES && V > 0 && V <= (1 << 24);
}

extern "C" int64_t mi355_verify_draft_workspace_bytes(int64_t num_seqs, int64_t num_nodes, int64_t vocab) {
  if (!vd_sizes_ok(num_seqs, num_nodes, vocab)) return 0;
  return num_seqs * (vd_rounds(num_nodes, vocab) * vd_pieces(vocab) * (int64_t)sizeof(double) + (int64_t)sizeof(int));
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
  const VdArgs a{target_probs, draft_probs, tokens, parents, uniforms, (int)num_nodes, (int)vocab, (int)vd_pieces(vocab), (int)vd_blocks(vocab)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int rounds = vd_rounds(num_nodes, vocab);
  double* sums = (double*)workspace;
  int* stop = (int*)(sums + rounds * num_seqs * a.pieces);
  // The first launch: about 512 workgroups, all resident.  The later ones: few sequences want them, with as many workgroups as
  // there are batches; the other sequences' cost one word each.
  int64_t batches = num_seqs * a.pieces / (VD_SUM_PIECES * 512);
  batches = batches < 1 ? 1 : batches > 16 ? 16 : batches;
  dim3 block(VD_SUM_THREADS);
  for (int round = 0; round < rounds; round++) {
    const int64_t per_wg = VD_SUM_PIECES * batches;
    dim3 grid((unsigned)((a.pieces + per_wg - 1) / per_wg), (unsigned)num_seqs);
    hipLaunchKernelGGL(verify_sums_kernel, grid, block, 0, s, a, sums, stop, round, (int)batches);
    if (int rc = check_launch("verify_sums_kernel", grid, block, 0)) return rc;
    batches = 1;
  }
  dim3 grid2((unsigned)num_seqs), block2(VD_WALK_THREADS);
  hipLaunchKernelGGL(verify_walk_kernel, grid2, block2, 0, s, a, (const double*)sums, (const int*)stop, rounds, path, num_accepted, next_token);
  return check_launch("verify_walk_kernel", grid2, block2, 0);
}
