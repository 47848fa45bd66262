// Attention of drafted token trees over a paged KV cache (the verification step of speculative decoding), head dim 128.
//
// Sequence s holds L = seq_lens[s] tokens, the last N of them its drafts, node n at position L - N + n.  A node's query
// sees every token in front of the drafts, itself and its ancestors.  With G query heads per kv head there are R = N * G
// query rows (row r: node r / G, head r % G of the group) that read the same keys and values: they share one pass.
//
// The op is HBM bound up to about 250 rows (a K and a V row are 512 bytes and 512 flop per query row; 1.29 PFLOP/s against 5 TB/s).
// Up to 32 rows are this file's kernel, built as the one-token decode kernel is: every wave streams its own steps of 32
// tokens -- K straight into MFMA operand registers, V through a private LDS ring by direct-to-LDS loads, both one step
// ahead -- and no wave waits for another before the end.  What differs: a step's K and V serve C = 1 or 2 column groups
// of 16 query rows, and scores of draft positions are masked by the node's set of ancestors, a 64-bit word per node made
// from the parents once per workgroup by pointer doubling.  More rows are the prefill kernel's TREE form, whose waves
// split the rows and share a tile: with four column groups here every wave read every V fragment for itself, and 64
// sequences of 512 to 8192 tokens with 64 rows took 317 us, on the TREE form 208 (and 175 with today's order of work).
//
// The longest sequence is cut into up to num_splits chunks of equally many 32-token steps, the others into chunks as long (see
// tree_chunk_steps); a sequence that fits one chunk writes its result directly, the others write fp32 partials that a second
// launch merges (two launches wherever num_splits > 1: the lengths are not known on the host).  Full chunks are handed out before
// shorter ones, see tree.hpp.
//
// Measured, 8 K/V heads: one sequence of 32768 tokens (28 rows, fp16) 33 us, of which the second launch is 5 (the first reads
// 5.1 TB/s); 64 of 512 to 8192 tokens (64 rows, bf16) 175 us, 4.3 TB/s.  Looking masked steps over for non-finite values is 1
// of the one and 5 of the other.
#include "tree.hpp"
#include <math.h>

namespace mi355 {

constexpr int PT_WAVES = 4;
constexpr int PT_WAVE_LDS = 2 * 8192;  // two stages of 32 V rows
constexpr int PT_ACC_ROW = 132;  // words per row of sums in the waves' merge: rows on the same banks took 1.4 us of a call
constexpr int PT_MAX_GROUP = 128;  // query heads per kv head

// bits 0 .. n - 1, at most four of them
__device__ __forceinline__ unsigned pt_first4(int n) { return n >= 4 ? 15u : n <= 0 ? 0u : (1u << n) - 1u; }

// The entries of v whose bit of `there` is set, zeros for the others and, unless the step is clean, for infinities and NaN.  By
// bit operations, as in tree_hide: conditional assignments to the vector's elements have been compiled to ones that keep them.
template <bool BF>
__device__ __forceinline__ half4 pt_keep(half4 v, unsigned there, bool clean) {
  uint2 w = __builtin_bit_cast(uint2, v);
  auto keep = [&](unsigned two, unsigned bits) {
    unsigned m = ((bits & 1u) | (bits & 2u) << 15) * 0xFFFFu;
    if (!clean) m &= ~((tree_nonfinite2<BF>(two) >> 15) * 0xFFFFu);
    return two & m;
  };
  w.x = keep(w.x, there), w.y = keep(w.y, there >> 2);
  return __builtin_bit_cast(half4, w);
}

template <int C, bool BF>
__global__ __launch_bounds__(PT_WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_tree_kernel(TreeArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, g = lane >> 4;
  const int reach = (a.max_pages << a.page_shift) * 16;
  const int kvh = blockIdx.x % a.num_kv_heads;
  int seq, split;
  const int chunk_steps = tree_chunk_steps(a.seq_lens, a.num_seqs, a.num_splits, a.per_half, reach);
  if (!tree_item(a.seq_lens, a.num_seqs, a.num_splits, chunk_steps, reach, blockIdx.x / a.num_kv_heads, seq, split)) return;
  const int R = a.nodes * a.group;
  const int num_q_heads = a.num_kv_heads * a.group;

  const int L_in = a.seq_lens[seq];
  const int L = L_in < 0 ? 0 : (L_in > reach ? reach : L_in);
  const int draft0 = L - a.nodes;  // position of node 0 (negative: the first nodes are not in the cache)
  const int steps = (L + 31) >> 5;
  const int s_begin = split * chunk_steps;
  const int s_end = s_begin + chunk_steps < steps ? s_begin + chunk_steps : steps;
  // a chunk behind the sequence's end has nothing to do; chunk 0 of an empty sequence writes its zeros
  if (s_begin >= steps && split > 0) return;
  const bool single = steps <= chunk_steps;
  const int p_end = (L + 15) >> 4;  // 16-token blocks
  const int n_steps = s_end - s_begin;

  unsigned long long* anc = reinterpret_cast<unsigned long long*>(lds);
  if (wave == 0) anc[lane] = tree_ancestors(a.parents + (size_t)seq * a.nodes, a.nodes);
  __syncthreads();
  unsigned long long seen[C];
  half8 qf[C][4];
#pragma unroll
  for (int c = 0; c < C; c++) {
    const int r = c * 16 + i16;
    const int node = r < R ? r / a.group : 0;
    const int head = kvh * a.group + (r < R ? r - node * a.group : 0);
    seen[c] = anc[node];
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
      if (r < R) {
        qf[c][ks] = *reinterpret_cast<const half8*>(a.q + (((size_t)seq * a.nodes + node) * num_q_heads + head) * 128 + ks * 32 + g * 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) qf[c][ks][e] = (half_t)0;
      }
    }
  }
  __syncthreads();  // the words are part of the V ring

  // page ids come through the scalar cache (constant address space: the table is not written while the kernel runs): a
  // vector load would have to be waited for in the order of the K and V loads in flight
  typedef const int __attribute__((address_space(4)))* table_ptr_t;
  const table_ptr_t bt = (table_ptr_t)(unsigned long long)(a.table + (size_t)seq * a.max_pages);
  char* my_lds = lds + wave * PT_WAVE_LDS;
  const size_t tok_stride = (size_t)a.num_kv_heads * 128;
  const half_t* k_lane = a.kc + (size_t)kvh * 128 + i16 * tok_stride + g * 8;
  const int vl_row = lane >> 4, vl_slot = lane & 15;
  const half_t* v_lane = a.vc + (size_t)kvh * 128 + vl_row * tok_stride;
  const int vr_row = 4 * g + (i16 >> 2);
  const int vr_base = vr_row * 256 + ((((i16 & 3) >> 1) ^ (2 * (vr_row & 7))) * 16) + (i16 & 1) * 8;  // ^ (dt * 32)

  half8 kf[2][2][4];  // [buffer][16-token block][ks]
  int bad[2] = {0, 0};  // bit x: block x of the step in this buffer has no page (its tokens are dropped)
  auto issue = [&](int step, int buf) {
    const int pa = 2 * (s_begin + wave + PT_WAVES * step);
    const int sub = (1 << a.page_shift) - 1;
    int id0 = bt[pa >> a.page_shift];
    int id1 = (pa + 1 < p_end) ? bt[(pa + 1) >> a.page_shift] : id0;
    const int drop0 = (unsigned)id0 >= (unsigned)a.num_pages, drop1 = (unsigned)id1 >= (unsigned)a.num_pages;
    id0 = drop0 ? 0 : id0;
    id1 = drop1 ? 0 : id1;
    bad[buf] = drop0 | (drop1 << 1);
    const size_t blk0 = ((size_t)id0 << a.page_shift) + (pa & sub);
    const size_t blk1 = (pa + 1 < p_end) ? ((size_t)id1 << a.page_shift) + ((pa + 1) & sub) : blk0;
    char* dst = my_lds + buf * 8192;
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const size_t off = (x ? blk1 : blk0) * 16 * tok_stride;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int chunk = vl_slot ^ (2 * ((4 * (i & 1) + vl_row) & 7));
        load_lds_16B(v_lane + off + (size_t)(4 * i) * tok_stride + chunk * 8, dst + x * 4096 + i * 1024);
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
      const size_t off = (x ? blk1 : blk0) * 16 * tok_stride;
#pragma unroll
      for (int ks = 0; ks < 4; ks++) kf[buf][x][ks] = *reinterpret_cast<const half8*>(k_lane + off + ks * 32);
    }
  };

  floatx4 oacc[C][8];
  float m_run[C], l_run[C];
#pragma unroll
  for (int c = 0; c < C; c++) {
    m_run[c] = -INFINITY, l_run[c] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 8; dt++) oacc[c][dt] = floatx4{0.f, 0.f, 0.f, 0.f};
  }

  const int my_steps = n_steps > wave ? (n_steps - wave + PT_WAVES - 1) / PT_WAVES : 0;
  if (my_steps > 0) issue(0, 0);
#pragma unroll 1
  for (int u = 0; u < my_steps; u += 2) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const int step = u + b;
      if (step < my_steps) {
        if (step + 1 < my_steps) {
          issue(step + 1, b ^ 1);
          asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const int pa = 2 * (s_begin + wave + PT_WAVES * step);
        const int tok0 = pa * 16 + 4 * g;  // lane (row i16, g) holds tokens tok0 + r and tok0 + 16 + r
        const bool drop0 = bad[b] & 1, drop1 = bad[b] & 2;
        const bool edge = pa * 16 + 32 > draft0 || bad[b] != 0;  // the step reaches into the drafts, past the end, or drops a block
        half8 pf[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
          floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < 4; ks++) s0 = mfma16_16x16x32<BF>(kf[b][0][ks], qf[c][ks], s0);
#pragma unroll
          for (int ks = 0; ks < 4; ks++) s1 = mfma16_16x16x32<BF>(kf[b][1][ks], qf[c][ks], s1);
          if (edge) {
            const unsigned vis0 = drop0 ? 0u : tree_visible4(seen[c], tok0 - draft0);
            const unsigned vis1 = drop1 ? 0u : tree_visible4(seen[c], tok0 + 16 - draft0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
              s0[r] = tree_hide(s0[r], vis0, r);
              s1[r] = tree_hide(s1[r], vis1, r);
            }
          }
          float mx = fmaxf(fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3])), fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3])));
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float m_new = fmaxf(m_run[c], mx);
          const bool none_yet = m_new == -INFINITY;
          const float alpha = none_yet ? 1.f : __builtin_amdgcn_exp2f((m_run[c] - m_new) * a.scale_log2e);
          const float mc = none_yet ? 0.f : m_new * a.scale_log2e;
          m_run[c] = m_new;
          // weights go into the second product in 16 bits, and the sum is that of the rounded ones: their error then is one of
          // weights that add up to 1, and the same as in the form with more rows
          float psum = 0.f;
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const half2v p0 = cvt16x2<BF>(__builtin_amdgcn_exp2f(s0[r] * a.scale_log2e - mc), __builtin_amdgcn_exp2f(s0[r + 1] * a.scale_log2e - mc));
            const half2v p1 = cvt16x2<BF>(__builtin_amdgcn_exp2f(s1[r] * a.scale_log2e - mc), __builtin_amdgcn_exp2f(s1[r + 1] * a.scale_log2e - mc));
            psum = dot2_ones<BF>(p1, dot2_ones<BF>(p0, psum));
            pf[c][r] = p0[0], pf[c][r + 1] = p0[1];
            pf[c][4 + r] = p1[0], pf[c][5 + r] = p1[1];
          }
          l_run[c] = l_run[c] * alpha + psum;
#pragma unroll
          for (int dt = 0; dt < 8; dt++) oacc[c][dt] = oacc[c][dt] * alpha;
        }
        const char* vst = my_lds + b * 8192;
        // What a query does not see does not reach it, whatever it holds: a weight of zero times a non-finite V entry would be
        // NaN.  In the steps with masked tokens such entries are added by themselves to the queries that see them (the
        // sums become infinity or NaN, whatever the weight) and left out of the product.
        bool clean = true;
        unsigned there0 = 15, there1 = 15;  // which of the lane's tokens are in the cache
        if (edge) {
          there0 = drop0 ? 0u : pt_first4(L - tok0);
          there1 = drop1 ? 0u : pt_first4(L - tok0 - 16);
          unsigned any = 0;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const uint4 x = *reinterpret_cast<const uint4*>(vst + (i * 64 + lane) * 16);
            any |= tree_nonfinite2<BF>(x.x) | tree_nonfinite2<BF>(x.y) | tree_nonfinite2<BF>(x.z) | tree_nonfinite2<BF>(x.w);
          }
          clean = __builtin_amdgcn_ballot_w64(any != 0) == 0;
          if (!clean) {
#pragma unroll 1
            for (int j = 0; j < 32; j++) {
              const int t = pa * 16 + j;
              if (t >= L || (j < 16 ? drop0 : drop1)) continue;
              unsigned sees[C];
#pragma unroll
              for (int c = 0; c < C; c++) sees[c] = 0u - (tree_visible4(seen[c], t - draft0) & 1u);
#pragma unroll
              for (int dt = 0; dt < 8; dt++) {
                const int row = j & 15, chunk = (2 * dt + (g >> 1)) ^ (2 * (row & 7));
                uint2 v = *reinterpret_cast<const uint2*>(vst + (j >> 4) * 4096 + row * 256 + chunk * 16 + (g & 1) * 8);
                v.x &= (tree_nonfinite2<BF>(v.x) >> 15) * 0xFFFFu, v.y &= (tree_nonfinite2<BF>(v.y) >> 15) * 0xFFFFu;
#pragma unroll
                for (int c = 0; c < C; c++) {
                  const unsigned x = v.x & sees[c], y = v.y & sees[c];
                  const floatx4 add = {tree_value<BF>(x & 0xFFFFu), tree_value<BF>(x >> 16), tree_value<BF>(y & 0xFFFFu), tree_value<BF>(y >> 16)};
                  oacc[c][dt] = oacc[c][dt] + add;
                }
              }
            }
          }
        }
#pragma unroll
        for (int dt = 0; dt < 8; dt++) {
          half4 lo = lds_read_tr16(vst + (vr_base ^ (dt * 32)));
          half4 hi = lds_read_tr16(vst + 4096 + (vr_base ^ (dt * 32)));
          if (edge) {  // 0 * garbage must stay 0
            lo = pt_keep<BF>(lo, there0, clean);
            hi = pt_keep<BF>(hi, there1, clean);
          }
          const half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
          for (int c = 0; c < C; c++) oacc[c][dt] = mfma16_16x16x32<BF>(vf, pf[c], oacc[c][dt]);
        }
      }
    }
  }

  // ---- merge the four waves through LDS, one column group at a time ----
  float* sm = reinterpret_cast<float*>(lds);  // [wave][16]
  float* sl = sm + PT_WAVES * 16;
  float* sacc = sl + PT_WAVES * 16;           // [wave][16][PT_ACC_ROW]
#pragma unroll
  for (int c = 0; c < C; c++) {
    float l = l_run[c] + __shfl_xor(l_run[c], 16);
    l += __shfl_xor(l, 32);
    __syncthreads();  // the V rings (or the group before) are done with
    if (g == 0) {
      sm[wave * 16 + i16] = m_run[c];
      sl[wave * 16 + i16] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; dt++) *reinterpret_cast<floatx4*>(sacc + ((wave * 16 + i16) * PT_ACC_ROW + dt * 16 + 4 * g)) = oacc[c][dt];
    __syncthreads();
#pragma unroll
    for (int idx = threadIdx.x; idx < 16 * 32; idx += PT_WAVES * 64) {  // 32 lanes of four columns per row
      const int col = idx >> 5, d = (idx & 31) * 4, r = c * 16 + col;
      if (r >= R) continue;
      float m_tot = -INFINITY;
#pragma unroll
      for (int w = 0; w < PT_WAVES; w++) m_tot = fmaxf(m_tot, sm[w * 16 + col]);
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
      float lt = 0.f;
#pragma unroll
      for (int w = 0; w < PT_WAVES; w++) {
        // (no maximum: zeros, or a row of scores that are not numbers; either is passed on as it is)
        const float wgt = m_tot > -INFINITY ? __builtin_amdgcn_exp2f((sm[w * 16 + col] - m_tot) * a.scale_log2e) : 1.f;
        const floatx4 p = *reinterpret_cast<const floatx4*>(sacc + (w * 16 + col) * PT_ACC_ROW + d);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(wgt, p[e], acc[e]);
        lt = __builtin_fmaf(wgt, sl[w * 16 + col], lt);
      }
      const int node = r / a.group;
      const size_t row = ((size_t)seq * a.nodes + node) * num_q_heads + kvh * a.group + (r - node * a.group);
      if (single) {
        const float inv = lt == 0.f ? 0.f : 1.f / lt;
        const half4 v = {cvt16<BF>(acc[0] * inv), cvt16<BF>(acc[1] * inv), cvt16<BF>(acc[2] * inv), cvt16<BF>(acc[3] * inv)};
        *reinterpret_cast<half4*>(a.out + row * 128 + d) = v;
      } else {
        const size_t at = row * a.num_splits + split;
        *reinterpret_cast<floatx4*>(a.part_acc + at * 128 + d) = acc;
        if (d == 0) {
          a.part_ml[at * 2] = m_tot * a.scale_log2e;
          a.part_ml[at * 2 + 1] = lt;
        }
      }
    }
  }
}

// Merge of the chunks of every row whose sequence has more than one.  A row's 128 sums are 32 lanes of 16 bytes, so that a
// group of 32 lanes takes a chunk at a time; GROUPS of them share a row's chunks and add up through LDS (few chunks: one group
// per row, eight rows per workgroup; many: the whole workgroup on one row, so that a row waits for memory
// num_splits / 8 times and not num_splits times).
template <bool BF, int GROUPS>
__global__ __launch_bounds__(256) void paged_tree_merge_kernel(TreeArgs a, int num_rows) {
  constexpr int ROWS = 8 / GROUPS;
  __shared__ floatx4 sum[8][32];
  __shared__ float weight[8];
  const int l32 = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int row = blockIdx.x * ROWS + grp / GROUPS, part = grp % GROUPS;
  const bool on = row < num_rows;
  const int seq = (on ? row : 0) / (a.nodes * a.num_kv_heads * a.group);
  const int reach = (a.max_pages << a.page_shift) * 16;
  const int L_in = a.seq_lens[seq];
  const int L = L_in < 0 ? 0 : (L_in > reach ? reach : L_in);
  const int steps = (L + 31) >> 5;
  const int chunk_steps = tree_chunk_steps(a.seq_lens, a.num_seqs, a.num_splits, a.per_half, reach);
  const int n = !on || steps <= chunk_steps ? 0 : (steps + chunk_steps - 1) / chunk_steps;
  const float* ml = a.part_ml + (size_t)row * a.num_splits * 2;
  const float* acc = a.part_acc + (size_t)row * a.num_splits * 128 + l32 * 4;
  float m_tot = -INFINITY;
  for (int s = l32; s < n; s += 32) m_tot = fmaxf(m_tot, ml[2 * s]);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m_tot = fmaxf(m_tot, __shfl_xor(m_tot, d));
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int s = part; s < n; s += GROUPS) {
    const float w = m_tot > -INFINITY ? __builtin_amdgcn_exp2f(ml[2 * s] - m_tot) : 1.f;  // (see the kernel's own merge)
    const floatx4 p = *reinterpret_cast<const floatx4*>(acc + (size_t)s * 128);
    l = __builtin_fmaf(w, ml[2 * s + 1], l);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(w, p[e], o[e]);
  }
  if constexpr (GROUPS > 1) {
    sum[grp][l32] = o;
    if (l32 == 0) weight[grp] = l;
    __syncthreads();
    if (grp % GROUPS) return;
#pragma unroll
    for (int k = 1; k < GROUPS; k++) {
      const floatx4 p = sum[grp + k][l32];
      l += weight[grp + k];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] += p[e];
    }
  }
  if (n == 0) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const half4 v = {cvt16<BF>(o[0] * inv), cvt16<BF>(o[1] * inv), cvt16<BF>(o[2] * inv), cvt16<BF>(o[3] * inv)};
  *reinterpret_cast<half4*>(a.out + (size_t)row * 128 + l32 * 4) = v;
}

template <bool BF, int GROUPS>
static int launch_merge(const TreeArgs& a, int64_t rows, hipStream_t stream) {
  dim3 grid((unsigned)((rows * GROUPS + 7) / 8)), block(256);
  hipLaunchKernelGGL((paged_tree_merge_kernel<BF, GROUPS>), grid, block, 0, stream, a, (int)rows);
  return check_launch("paged_tree_merge_kernel", grid, block, 0);
}

template <int C, bool BF>
static int launch_tree(const TreeArgs& a, int num_seqs, hipStream_t stream) {
  auto kern = paged_tree_kernel<C, BF>;
  constexpr int lds_bytes = PT_WAVES * PT_WAVE_LDS;
  static_assert(lds_bytes >= (int)((2 * PT_WAVES * 16 + PT_WAVES * 16 * PT_ACC_ROW) * sizeof(float)), "merge area must fit");
  static std::atomic<uint64_t> lds_ok{0};
  if (int rc = allow_lds(reinterpret_cast<const void*>(kern), lds_bytes, lds_ok, "paged_tree_kernel")) return rc;
  const int64_t wgs = (int64_t)num_seqs * a.num_splits * a.num_kv_heads;
  if (wgs >= (1ll << 24)) return fail(-MI355_E_SHAPE, "paged_tree_attn: too many workgroups");  // 2^32 threads
  dim3 grid((unsigned)wgs), block(PT_WAVES * 64);
  hipLaunchKernelGGL(kern, grid, block, lds_bytes, stream, a);
  return check_launch("paged_tree_kernel", grid, block, lds_bytes);
}

template <bool BF>
static int run_tree(TreeArgs a, int num_seqs, hipStream_t stream) {
  const int R = a.nodes * a.group;
  int rc;
  if (R <= 16) rc = launch_tree<1, BF>(a, num_seqs, stream);
  else if (R <= 32) rc = launch_tree<2, BF>(a, num_seqs, stream);
  else rc = fa_tree(a, num_seqs, BF, stream);
  if (rc || a.num_splits == 1) return rc;
  const int64_t rows = (int64_t)num_seqs * R * a.num_kv_heads;
  return a.num_splits <= 8 ? launch_merge<BF, 1>(a, rows, stream) : launch_merge<BF, 8>(a, rows, stream);
}

}  // namespace mi355

using namespace mi355;

// At most 64 chunks, and no more than a full table has 128-token ones, for about so many workgroups: 256 where few (sequence, K/V head, 128 rows) blocks read
// long caches on the kernel above, which a workgroup per CU drives at memory's rate (one sequence of 32768 tokens 36 / 31 / 35 us
// with 128 / 256 / 384 workgroups), 512 where the prefill form does, which needs two per CU (64 rows: 41 / 37 with 256 / 384), or
// with 20 to 32 blocks; more blocks differ in length, and 1024 in order of their size even that out (64 sequences of
// 512-8192 tokens with 64 rows 231 / 170 / 175 / 206 us with 512 / 1024 / 1536 / 4096, 8 of 1000-16384 63 / 51 / 62 with 512 / 1024 / 1536).
extern "C" int64_t mi355_paged_tree_default_splits(int64_t num_seqs, int64_t num_nodes, int64_t num_q_heads, int64_t num_kv_heads,
                                                   int64_t page_size, int64_t max_pages_per_seq) {
  if (num_seqs <= 0 || num_nodes <= 0 || num_q_heads <= 0 || num_kv_heads <= 0) return 1;
  const int64_t rows = num_nodes * num_q_heads / num_kv_heads, blocks = num_seqs * num_kv_heads * ((rows + 127) / 128);
  if (blocks <= 0 || blocks > 1024) return 1;
  const int64_t wgs = blocks > 32 ? 1024 : blocks >= 20 || rows > 32 ? 512 : 256;
  const int64_t fill = wgs / blocks, tokens = max_pages_per_seq * page_size / 128, n = fill < tokens ? fill : tokens;
  return n < 1 ? 1 : n > 64 ? 64 : n;
}

extern "C" int mi355_paged_tree_attn(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                     const int32_t* seq_lens, const int32_t* parents, void* out, float* part_acc, float* part_ml,
                                     int64_t num_seqs, int64_t num_nodes, int64_t num_q_heads, int64_t num_kv_heads, int64_t D,
                                     int64_t page_size, int64_t max_pages_per_seq, int64_t num_pages, int64_t num_splits, float scale,
                                     int dtype, void* stream) {
  const char* fn = "paged_tree_attn";
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !parents || !out) return fail(-MI355_E_NULL, "%s: null pointer", fn);
  if (dtype != MI355_F16 && dtype != MI355_BF16) return fail(-MI355_E_DTYPE, "%s: dtype %d (MI355_F16 or MI355_BF16)", fn, dtype);
  if (D != 128) return fail(-MI355_E_SHAPE, "%s: head dim %lld not supported (only 128)", fn, (long long)D);
  int page_shift = -1;
  for (int sh = 0; sh <= 4; sh++)
    if (page_size == (16ll << sh)) page_shift = sh;
  if (page_shift < 0) return fail(-MI355_E_SHAPE, "%s: page size %lld not supported (16, 32, 64, 128 or 256)", fn, (long long)page_size);
  if (num_nodes <= 0 || num_nodes > TREE_MAX_NODES)
    return fail(-MI355_E_SHAPE, "%s: %lld nodes per sequence, supported: 1 to %d", fn, (long long)num_nodes, TREE_MAX_NODES);
  if (num_seqs <= 0 || num_seqs > 65535 || num_q_heads <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_q_heads > 65535 ||
      max_pages_per_seq <= 0 || max_pages_per_seq > (1 << 22) || num_pages <= 0 || num_pages > (1 << 26) ||
      num_seqs * num_nodes * num_q_heads > (num_splits > 1 ? 1ll << 23 : 1ll << 30) || max_pages_per_seq * page_size > (1ll << 30))
    return fail(-MI355_E_SHAPE, "%s: bad sizes seqs=%lld nodes=%lld hq=%lld hkv=%lld max_pages=%lld num_pages=%lld", fn,
                (long long)num_seqs, (long long)num_nodes, (long long)num_q_heads, (long long)num_kv_heads,
                (long long)max_pages_per_seq, (long long)num_pages);
  if (num_q_heads % num_kv_heads != 0)
    return fail(-MI355_E_SHAPE, "%s: q heads %lld not a multiple of kv heads %lld", fn, (long long)num_q_heads, (long long)num_kv_heads);
  if (num_q_heads / num_kv_heads > PT_MAX_GROUP)
    return fail(-MI355_E_SHAPE, "%s: q heads per kv head = %lld, supported: up to %d", fn, (long long)(num_q_heads / num_kv_heads), PT_MAX_GROUP);
  if (num_splits < 1 || num_splits > 1024) return fail(-MI355_E_SHAPE, "%s: num_splits %lld out of range [1, 1024]", fn, (long long)num_splits);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be positive and finite", fn);
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return fail(-MI355_E_ALIGN, "%s: q, k_cache, v_cache, out must be 16-byte aligned", fn);
  if (num_splits > 1 && (!part_acc || !part_ml)) return fail(-MI355_E_SCRATCH, "%s: num_splits > 1 needs part_acc / part_ml scratch", fn);
  if (num_splits > 1 && !aligned16(part_acc)) return fail(-MI355_E_ALIGN, "%s: part_acc must be 16-byte aligned", fn);
  TreeArgs a{(const half_t*)q, (const half_t*)k_cache, (const half_t*)v_cache, block_table, seq_lens, parents, (half_t*)out,
           part_acc, part_ml, (int)num_kv_heads, (int)(num_q_heads / num_kv_heads), (int)num_nodes, (int)max_pages_per_seq,
           (int)num_pages, page_shift, (int)num_splits, (int)num_seqs, tree_per_half(num_splits), scale * 1.4426950408889634f};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return dtype == MI355_BF16 ? run_tree<true>(a, (int)num_seqs, s) : run_tree<false>(a, (int)num_seqs, s);
}
