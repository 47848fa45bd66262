// Flash-attention forward (prefill) for gfx950, head dim 128, fp16 in/out, fp32 softmax.
//
// One workgroup = 4 waves = 128 queries of one (batch, head); each wave owns 32 queries and
// keeps, in registers, its Q fragments (32 VGPRs), the running max / sum of every query, and
// the 32 x 128 fp32 output accumulator (64 VGPRs).  K and V are streamed in 64-key tiles
// through a two-stage LDS ring filled by direct-to-LDS loads.
//
// Both contractions are computed transposed so that the softmax never leaves registers:
//   S^T[key][query]  = K . Q^T     (MFMA A operand = K rows from LDS, B operand = Q in registers)
//   O^T[d][query]   += V^T . P^T   (A operand = V^T via LDS transpose reads, B operand = P)
// With v_mfma_f32_32x32x16_f16 a lane owns one query column of S^T (16 keys per 32-key tile,
// the other 16 sit in lane^32), so row max / sum are in-lane reductions plus one cross-lane
// exchange, and the exponentiated scores are already laid out as the B operand of the second
// MFMA.  The order in which keys are fed to that MFMA is whatever the S^T register order
// dictates; V^T is fetched with the matching order by ds_read_b64_tr_b16.
//
// LDS swizzles (16-byte chunks, 256-byte rows): K chunk c of row r -> slot c ^ (r & 15);
// V chunk c of row r -> slot c ^ (2 * (r & 7)).  As in the GEMM, the swizzle is applied on the
// global side of the direct-to-LDS loads.
#include "common.hpp"
#include "tree.hpp"
#include <math.h>
#include <type_traits>

namespace mi355 {

constexpr int FA_BLOCK_M = 128;
constexpr int FA_BLOCK_N = 64;
constexpr int FA_STAGE = 2 * FA_BLOCK_N * 256;  // K tile + V tile, bytes

// Where each operand's (batch, head, row) lives, in elements; the 128 elements of a row are contiguous.
// `group` query heads share one K/V head (1 = plain multi-head attention).
struct FaLayout {
  int64_t q_b, q_h, k_b, k_h, v_b, v_h, o_b, o_h;
  unsigned q_r, k_r, v_r, o_r;
  int H, group;
};

template <bool CAUSAL, bool BF>
__global__ __launch_bounds__(256) void fa_fwd_d128(const half_t* __restrict__ Q, const half_t* __restrict__ K,
                                                   const half_t* __restrict__ V, half_t* __restrict__ O, int BH, int Sq,
                                                   int Sk, float scale_log2e, int q_blocks, FaLayout lay) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;

  // workgroup -> (batch*head, query block).  Consecutive ids land on different XCDs; keep all
  // query blocks of one head on one XCD so its K/V stay in that XCD's L2.
  int bh, qb;
  {
    const int pid = blockIdx.x;
    if (((BH / lay.group) & 7) == 0) {
      // all query blocks of the `group` query heads that share one K/V head sit on one XCD
      const int xcd = pid & 7, loc = pid >> 3, per_kv = q_blocks * lay.group;
      const int w = loc % per_kv;
      bh = ((loc / per_kv) * 8 + xcd) * lay.group + w / q_blocks;
      qb = w % q_blocks;
    } else {
      bh = pid / q_blocks;
      qb = pid % q_blocks;
    }
    if (CAUSAL) qb = q_blocks - 1 - qb;  // longest rows first
  }
  const int causal_off = Sk - Sq;  // query i sees keys <= i + causal_off
  const int q0 = qb * FA_BLOCK_M;
  const int wq0 = q0 + wave * 32;  // first query of this wave
  const int q_row = wq0 + r32;
  const bool q_ok = q_row < Sq;

  const int b_idx = bh / lay.H, h_idx = bh - b_idx * lay.H, hk_idx = h_idx / lay.group;
  const half_t* Qb = Q + b_idx * lay.q_b + h_idx * lay.q_h;
  const half_t* Kb = K + b_idx * lay.k_b + hk_idx * lay.k_h;
  const half_t* Vb = V + b_idx * lay.v_b + hk_idx * lay.v_h;
  half_t* Ob = O + b_idx * lay.o_b + h_idx * lay.o_h;

  // number of key tiles this workgroup walks
  int k_end = Sk;
  if (CAUSAL) {
    int last_q = q0 + FA_BLOCK_M - 1;
    if (last_q > Sq - 1) last_q = Sq - 1;
    int lim = last_q + causal_off + 1;
    if (lim < k_end) k_end = lim;
  }
  const int n_tiles = k_end > 0 ? (k_end + FA_BLOCK_N - 1) / FA_BLOCK_N : 0;

  // ---- Q fragments (MFMA B operand): lane (query r32, half h) holds d = 16*ks + 8*h .. +7 ----
  half8 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) {
    if (q_ok) {
      qf[ks] = *reinterpret_cast<const half8*>(Qb + (size_t)q_row * lay.q_r + ks * 16 + h * 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) qf[ks][e] = (half_t)0;
    }
  }

  // ---- global -> LDS: a wave-load moves 4 rows of 256 bytes; lane l: row l/16, slot l%16 ----
  const int lrow = lane >> 4, lslot = lane & 15;
  const int k_chunk = lslot ^ (wave * 4 + lrow);           // group g = wave + 4*i, so (row & 15) = 4*wave + lrow
  const int v_chunk = lslot ^ (2 * ((wave & 1) * 4 + lrow));  // (row & 7) = 4*(wave&1) + lrow
  auto issue_loads = [&](int tile, int stage) {
    char* dst = lds + stage * FA_STAGE + wave * 1024;
    const int key0 = tile * FA_BLOCK_N;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      int row = key0 + (wave + 4 * i) * 4 + lrow;
      if (row > Sk - 1) row = Sk - 1;  // clamp: the tail rows are masked out of the softmax
      load_lds_16B(Kb + (size_t)row * lay.k_r + k_chunk * 8, dst + i * 4096);
      load_lds_16B(Vb + (size_t)row * lay.v_r + v_chunk * 8, dst + FA_BLOCK_N * 256 + i * 4096);
    }
  };

  // ---- LDS read addresses ----
  const int k_base = r32 * 256 + ((h ^ (lane & 15)) * 16);  // ^ (ks*32), + t*8192
  const int i16 = lane & 15, g16 = lane >> 4;
  const int v_row = 4 * (g16 >> 1) + (i16 >> 2);
  const int v_cl = 2 * (g16 & 1) + ((i16 & 3) >> 1);
  const int v_base = FA_BLOCK_N * 256 + v_row * 256 + ((v_cl ^ (2 * (v_row & 7))) * 16) + (i16 & 1) * 8;  // ^ (dt*64), + t16*4096, + {0,2048}

  floatx16 oacc[4];
#pragma unroll
  for (int dt = 0; dt < 4; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[dt][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  if (n_tiles > 0) {
    issue_loads(0, 0);
    wait_vmcnt0();
    __syncthreads();
  }

  for (int j = 0; j < n_tiles; j++) {
    if (j + 1 < n_tiles) issue_loads(j + 1, (j + 1) & 1);
    const char* st = lds + (j & 1) * FA_STAGE;
    const int key0 = j * FA_BLOCK_N;
    // a wave whose every query is before this tile has nothing to do here (causal only)
    const bool active = !CAUSAL || (key0 <= wq0 + 31 + causal_off);
    if (active) {
      floatx16 s[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
#pragma unroll
        for (int r = 0; r < 16; r++) s[t][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
          half8 kf = *reinterpret_cast<const half8*>(st + ((k_base ^ (ks * 32)) + t * 8192));
          s[t] = mfma16<BF>(kf, qf[ks], s[t]);
        }
      }
      const bool need_mask = (CAUSAL && (key0 + FA_BLOCK_N - 1 > wq0 + causal_off)) || (key0 + FA_BLOCK_N > Sk);
      if (need_mask) {
        const int lim = CAUSAL ? (q_row + causal_off < Sk - 1 ? q_row + causal_off : Sk - 1) : Sk - 1;  // last visible key
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int key = key0 + 32 * t + 8 * (r >> 2) + 4 * h + (r & 3);
            if (key > lim) s[t][r] = -INFINITY;
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[t][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_run, mx);
      const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
      const float alpha = exp2f((m_run - m_use) * scale_log2e);
      const float mc = m_use * scale_log2e;
      m_run = m_new;
      float psum = 0.f;
      half8 pf[4];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float p = exp2f(s[t][r] * scale_log2e - mc);
          psum += p;
          pf[t * 2 + (r >> 3)][r & 7] = cvt16<BF>(p);
        }
      l_run = l_run * alpha + psum;
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[dt][r] *= alpha;
      // O^T += V^T P^T
#pragma unroll
      for (int t16 = 0; t16 < 4; t16++) {
#pragma unroll
        for (int dt = 0; dt < 4; dt++) {
          const char* va = st + ((v_base ^ (dt * 64)) + t16 * 4096);
          half4 lo = lds_read_tr16(va);
          half4 hi = lds_read_tr16(va + 2048);
          half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          oacc[dt] = mfma16<BF>(vf, pf[t16], oacc[dt]);
        }
      }
    }
    wait_vmcnt0();
    __syncthreads();
  }

  // ---- epilogue ----
  const float l_tot = l_run + __shfl_xor(l_run, 32);
  const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
  if (q_ok) {
    half_t* orow = Ob + (size_t)q_row * lay.o_r + 4 * h;
#pragma unroll
    for (int dt = 0; dt < 4; dt++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        half4 v = {cvt16<BF>(oacc[dt][4 * q] * inv), cvt16<BF>(oacc[dt][4 * q + 1] * inv), cvt16<BF>(oacc[dt][4 * q + 2] * inv),
                   cvt16<BF>(oacc[dt][4 * q + 3] * inv)};
        *reinterpret_cast<half4*>(orow + dt * 32 + q * 8) = v;
      }
  }
}

// Paged K/V (the PAGED form of fa_fwd_d128_m16): the keys and values of sequence b are the first seq_lens[b] token rows of the
// pages block_table[b][0..], 16 << page_shift tokens per page, laid out [page][token][kv head][128].  The kernel
// walks 16-token blocks; a page is 1 << page_shift consecutive blocks.
struct FaPaged {
  const int* block_table;  // [batch][max_pages]
  const int* seq_lens;     // [batch]
  int max_pages, num_pages, page_shift;
};

// body(std::integral_constant<int, 0>{}), ..., body(std::integral_constant<int, N - 1>{}): a loop whose index is a
// constant expression in the body (instruction immediates of inline assembly need one).
template <int I, int N, typename F>
__device__ __forceinline__ void static_for(F&& body) {
  if constexpr (I < N) {
    body(std::integral_constant<int, I>{});
    static_for<I + 1, N>(body);
  }
}

// Software-pipelined form.  Same tiling and register layout, but the score MFMAs run one key tile
// ahead of the softmax: in trip j a wave issues S^T(j+1) = K(j+1) . Q^T, exponentiates the scores of
// tile j on the VALU while those MFMAs execute, then issues O^T += V(j)^T . P(j)^T.  K and V sit in
// separate two-deep LDS rings, K one tile ahead of V; the trip is written twice (scores ping-pong
// between two register sets, ring slots become compile-time constants) so nothing is copied.
// The running maximum is only raised -- and O rescaled -- when some query's maximum grew by more than
// 2^8; until then exponentials are taken against the stale maximum (they stay below 2^8, and O / l is
// the same quotient), which keeps the 64-register rescale off the common path.
// V swizzle: chunk c of row r -> slot c ^ (4 * (r & 3)), which keeps the four 64-byte row pieces that a
// half-wave transpose read touches on distinct banks (measured conflict-free; c ^ 2(r & 7) is not).
// NW = waves per workgroup: 4 (128 queries, two workgroups per CU) or 8 (256 queries, one workgroup per CU: the two
// wave quartets of a CU then share ONE copy of every K / V tile instead of loading one each -- half the LDS writes
// and half the L2 reads for the same fragment reads).
template <bool CAUSAL, bool BF, int NW = 4>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fa_fwd_d128_pipe(
    const half_t* __restrict__ Q, const half_t* __restrict__ K, const half_t* __restrict__ V, half_t* __restrict__ O, int BH,
    int Sq, int Sk, float scale_log2e, int q_blocks, FaLayout lay) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  static_assert(NW == 4 || NW == 8, "four or eight waves");
  constexpr int BLOCK_M = NW * 32;          // queries per workgroup
  constexpr int NI = 16 / NW;               // wave-loads per wave and tile (a wave-load = 4 rows of 256 bytes)
  constexpr int TILE_B = FA_BLOCK_N * 256;  // bytes of one K or V tile
  // (A three-slot ring for the 8-wave form -- tiles loaded two trips ahead, a trip waiting only for the loads of the
  // trip before -- measured 5 % slower than two slots: load latency is not what the trips wait for, and ring slots
  // that are not compile-time constants cost address arithmetic.)
  constexpr int VBUF = 2 * TILE_B;          // K ring at 0, V ring behind it
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;

  // Workgroup -> (batch * head, unit).  A unit is one 128-query block; with the causal mask it is a pair of
  // blocks, the i-th from the end and the i-th from the start, processed one after the other, so that every
  // workgroup walks the same number of key tiles (q_blocks + 1) and the grid has no long tail.
  const int units = CAUSAL ? (q_blocks + 1) / 2 : q_blocks;
  int bh, unit;
  {
    const int pid = blockIdx.x;
    if (((BH / lay.group) & 7) == 0) {
      // all units of the `group` query heads that share one K/V head sit on one XCD
      const int xcd = pid & 7, loc = pid >> 3, per_kv = units * lay.group;
      const int w = loc % per_kv;
      bh = ((loc / per_kv) * 8 + xcd) * lay.group + w / units;
      unit = w % units;
    } else {
      bh = pid / units;
      unit = pid % units;
    }
  }
  const int b_idx = bh / lay.H;
  const int h_idx = bh - b_idx * lay.H, hk_idx = h_idx / lay.group;
  const int causal_off = Sk - Sq;
  const half_t* Qb = Q + b_idx * lay.q_b + h_idx * lay.q_h;
  const half_t* Kb = K + b_idx * lay.k_b + hk_idx * lay.k_h;
  const half_t* Vb = V + b_idx * lay.v_b + hk_idx * lay.v_h;
  half_t* Ob = O + b_idx * lay.o_b + h_idx * lay.o_h;

  // LDS addresses of the eight K fragment reads of a 32-key half tile (ks = 0..7), formed once: left to the
  // compiler inside the pass loop, the offsets are hoisted as integers and each read then adds the LDS base to
  // one again, vector instructions that upset the pinned MFMA / softmax interleave
  typedef const __attribute__((address_space(3))) half8* lds_half8_t;
  unsigned k_frag[8];
  {
    const int kb0 = r32 * 256 + ((h ^ (lane & 15)) * 16);
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      k_frag[ks] = (unsigned)(uintptr_t)MI355_LDS(char, lds + (kb0 ^ (ks * 32)));
      asm volatile("" : "+v"(k_frag[ks]));  // one opaque value per read: nothing to re-derive it from
    }
  }
  // LDS addresses of the V^T transpose reads (slot 0 of the V ring; dt = 0..3), same treatment
  unsigned v_frag[4];
  {
    const int i16 = lane & 15, g16 = lane >> 4;
    const int v_row = 4 * (g16 >> 1) + (i16 >> 2);
    const int vb0 = VBUF + v_row * 256 + (i16 >> 2) * 64 + (2 * (g16 & 1) + ((i16 & 3) >> 1)) * 16 + (i16 & 1) * 8;
#pragma unroll
    for (int dt = 0; dt < 4; dt++) {
      v_frag[dt] = (unsigned)(uintptr_t)MI355_LDS(char, lds + (vb0 ^ (dt * 64)));
      asm volatile("" : "+v"(v_frag[dt]));
    }
  }
  for (int pass = 0; pass < (CAUSAL ? 2 : 1); pass++) {
  const int qb = CAUSAL ? (pass == 0 ? q_blocks - 1 - unit : unit) : unit;
  if (CAUSAL && pass == 1 && 2 * unit == q_blocks - 1) break;  // the middle block of an odd count has no partner
  const int q0 = qb * BLOCK_M;
  const int wq0 = q0 + wave * 32;
  const int q_row = wq0 + r32;
  const bool q_ok = q_row < Sq;

  int k_end = Sk;
  if (CAUSAL) {
    int last_q = q0 + BLOCK_M - 1;
    if (last_q > Sq - 1) last_q = Sq - 1;
    int lim = last_q + causal_off + 1;
    if (lim < k_end) k_end = lim;
  }
  const int n_tiles = k_end > 0 ? (k_end + FA_BLOCK_N - 1) / FA_BLOCK_N : 0;

  half8 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) {
    if (q_ok) {
      // scale . log2(e) is folded into Q (rounded to the 16-bit format again: a relative error of 2^-11 per
      // element for fp16, 2^-8 for bf16 -- the same size as the rounding of P), so the MFMA delivers exponents of
      // 2 directly
      const half8 raw = *reinterpret_cast<const half8*>(Qb + (size_t)q_row * lay.q_r + ks * 16 + h * 8);
#pragma unroll
      for (int e = 0; e < 8; e++) qf[ks][e] = cvt16<BF>(to_f32<BF>(raw[e]) * scale_log2e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) qf[ks][e] = (half_t)0;
    }
  }

  const int lrow = lane >> 4, lslot = lane & 15;
  const int k_chunk = lslot ^ ((wave * 4 + lrow) & 15);
  const int v_chunk = lslot ^ (4 * lrow);
  // Global -> LDS through a buffer descriptor rebuilt per tile on the scalar unit (base = first row of the tile,
  // size = up to the end of the tile's last valid row): the per-lane byte offset is loop-invariant, rows at or
  // beyond Sk read zeros (they are masked out of the softmax), and no 64-bit vector address arithmetic is left.
  const unsigned k_rb = lay.k_r * 2, v_rb = lay.v_r * 2;  // row strides in bytes
  const unsigned k_voff = (wave * 4 + lrow) * k_rb + k_chunk * 16;
  const unsigned v_voff = (wave * 4 + lrow) * v_rb + v_chunk * 16;
  auto issue_kv = [&](const half_t* base, unsigned rb, unsigned voff, int tile, int lds_off) {
    char* dst = lds + lds_off + wave * 1024;
    const int row0 = tile * FA_BLOCK_N;
    int rem = Sk - row0;
    rem = rem > FA_BLOCK_N ? FA_BLOCK_N : rem;
    const buffer_rsrc_t rs = make_buffer(reinterpret_cast<const char*>(base) + (size_t)row0 * rb, (unsigned)(rem - 1) * rb + 256u);
#pragma unroll
    for (int i = 0; i < NI; i++) buffer_load_lds_16B(rs, voff + (unsigned)(i * NW * 4) * rb, 0, dst + i * NW * 1024);
  };

  floatx16 oacc[4];
#pragma unroll
  for (int dt = 0; dt < 4; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[dt][r] = 0.f;
  // The running maximum m of a query lives negated in all 16 registers of `negm`, which every score MFMA chain
  // starts from: the accumulators then hold log2-domain scores relative to m and feed v_exp_f32 unchanged.
  // (A lane owns one query column of S^T, so the 16 values of a lane are equal.)
  floatx16 negm;
#pragma unroll
  for (int r = 0; r < 16; r++) negm[r] = 0.f;
  float l_run = 0.f;
  // m is raised -- and O rescaled -- only when a score exceeds it by more than 2^8; -inf until the query has
  // seen its first unmasked key, so that the first one always sets m
  float grow_thr = -INFINITY;
  constexpr float kRescaleThreshold = 8.f;

  auto wave_active = [&](int tile) { return !CAUSAL || (tile * FA_BLOCK_N <= wq0 + 31 + causal_off); };

  // S^T = K(slot) . Q^T, 16 MFMAs
  auto scores = [&](int koff, floatx16* s) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (int ks = 0; ks < 8; ks++) {
        half8 kf = *(lds_half8_t)(uintptr_t)(k_frag[ks] + (unsigned)(koff + t * 8192));
        s[t] = mfma16<BF>(kf, qf[ks], ks == 0 ? negm : s[t]);
      }
    }
  };

  // softmax of tile `tile` (scores in s) and O^T += V(slot)^T . P^T
  auto softmax_pv = [&](auto masked_tag, int tile, auto voff_tag, floatx16* s, int koff_next, floatx16* s_next) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    constexpr int VOFF = decltype(voff_tag)::value;  // byte offset of the V ring slot to read
    if (MASKED) {
      const int key0 = tile * FA_BLOCK_N;
      const bool need_mask = (CAUSAL && (key0 + FA_BLOCK_N - 1 > wq0 + causal_off)) || (key0 + FA_BLOCK_N > Sk);
      if (need_mask) {
        const int lim = CAUSAL ? (q_row + causal_off < Sk - 1 ? q_row + causal_off : Sk - 1) : Sk - 1;
        const int rel = lim - key0 - 4 * h;  // last visible key, relative to the tile and to this lane's rows
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 16; r++)
          {
            // -inf where the key is beyond `rel`, by bit selection: a compare-and-select per score would hold
            // a scalar register pair per score and push loop-invariant scalars out of the register file
            const unsigned hide = (unsigned)((rel - (32 * t + 8 * (r >> 2) + (r & 3))) >> 31);
            const float sv = s[t][r];  // (bit_cast straight from a vector element miscompiles)
            s[t][r] = __builtin_bit_cast(float, (hide & 0xFF800000u) | (~hide & __builtin_bit_cast(unsigned, sv)));
          }
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[t][r]);
    if (__builtin_amdgcn_ballot_w64(mx > grow_thr) != 0) {
      // rare: some query's scores outgrew its maximum (or it saw its first key).  The other half of a query's
      // keys sits in lane ^ 32; both lanes take the same decision.
      const float mxx = fmaxf(mx, __shfl_xor(mx, 32));
      const bool fresh = grow_thr == -INFINITY;
      const float delta = fresh ? (mxx == -INFINITY ? 0.f : mxx) : fmaxf(mxx, 0.f);
      const float alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(-delta);
      if (mxx != -INFINITY) grow_thr = kRescaleThreshold;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[dt][r] *= alpha;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) s[t][r] -= delta;
#pragma unroll
      for (int r = 0; r < 16; r++) negm[r] -= delta;
    }
    half8 pf[4];
    float psum = 0.f;
    // Scores of the next tile and exponentials of this one in one straight-line block: a wave issues in
    // order, so only VALU work placed between two MFMAs runs while the first occupies the matrix pipe.
    // (Past the last tile the scores are computed from stale LDS bytes and never used.)
    __builtin_amdgcn_sched_barrier(0);
    scores(koff_next, s_next);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const half2v pp = cvt16x2<BF>(__builtin_amdgcn_exp2f(s[t][r]), __builtin_amdgcn_exp2f(s[t][r + 1]));
        psum = dot2_ones<BF>(pp, psum);  // sums what the second MFMA multiplies
        pf[t * 2 + (r >> 3)][r & 7] = pp[0];
        pf[t * 2 + (r >> 3)][(r & 7) + 1] = pp[1];
      }
    // order: 3 K fragment reads up front, then per score MFMA one more read and the work of two scores
    // (two exp, one cvt_pk, one dot2) -- a fragment is requested two MFMAs before its use
    __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
    for (int i = 0; i < 13; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < 3; i++) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  
    l_run += psum;
    // O^T += V^T P^T: 16 MFMAs, each V^T fragment (two transpose reads) requested two MFMAs ahead.
    // The reads and their waits are inline assembly: a transpose read the compiler can see makes it wait for
    // EVERY direct-to-LDS load in flight first (it cannot tell that the loads fill other ring slots), which put a
    // vmcnt(0) -- the loads issued at the head of this trip -- in the middle of every trip.  In this block nothing
    // else counts in lgkmcnt: LDS returns in order, so MFMA i may run once at most the reads of fragments i + 1
    // and i + 2 (two each) are outstanding.  Each wait names the fragment's registers, so no use moves above it.
    half4 vlo[3], vhi[3];
    auto vr = [&](auto itag) {  // i = t16*4 + dt
      constexpr int i = decltype(itag)::value;
      constexpr int off = VOFF + (i >> 2) * 4096;
      half4 &lo = vlo[i % 3], &hi = vhi[i % 3];  // (operands of an assembly statement do not capture by themselves)
      const unsigned addr = v_frag[i & 3];
      asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                   : "=&v"(lo), "=&v"(hi)
                   : "v"(addr), "n"(off), "n"(off + 2048));
    };
    vr(std::integral_constant<int, 0>{});
    vr(std::integral_constant<int, 1>{});
    static_for<0, 16>([&](auto itag) {
      constexpr int i = decltype(itag)::value;
      if constexpr (i + 2 < 16) vr(std::integral_constant<int, i + 2>{});
      half4 &lo = vlo[i % 3], &hi = vhi[i % 3];
      if constexpr (i + 2 < 16)
        asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(lo), "+v"(hi));
      else if constexpr (i + 1 < 16)
        asm volatile("s_waitcnt lgkmcnt(2)" : "+v"(lo), "+v"(hi));
      else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(lo), "+v"(hi));
      const half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      oacc[i & 3] = mfma16<BF>(vf, pf[i >> 2], oacc[i & 3]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  floatx16 sa[2], sb[2];
  if (n_tiles > 0) {
    issue_kv(Kb, k_rb, k_voff, 0, 0);
    issue_kv(Vb, v_rb, v_voff, 0, VBUF);
    if (n_tiles > 1) issue_kv(Kb, k_rb, k_voff, 1, TILE_B);
    wait_vmcnt0();
    __syncthreads();
    if (wave_active(0)) scores(0, sa);
    // trip 0 overwrites the K(0) slot with K(2): every wave must have read its K(0) fragments first
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // trip j (PAR = j & 1): loads for K(j+2) and V(j+1); scores of tile j+1; softmax + PV of tile j
  auto trip = [&](auto par_tag, int j, floatx16* s_cur, floatx16* s_next) {
    constexpr int PAR = decltype(par_tag)::value;
    constexpr int K_CUR = PAR * TILE_B, K_NEXT = (1 - PAR) * TILE_B, V_CUR = PAR * TILE_B, V_NEXT = VBUF + (1 - PAR) * TILE_B;
    if (j + 2 < n_tiles) issue_kv(Kb, k_rb, k_voff, j + 2, K_CUR);
    if (j + 1 < n_tiles) issue_kv(Vb, v_rb, v_voff, j + 1, V_NEXT);
    if (wave_active(j)) softmax_pv(std::true_type{}, j, std::integral_constant<int, V_CUR>{}, s_cur, K_NEXT, s_next);  // idle from here on otherwise
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
  };
  for (int j = 0; j < n_tiles; j += 2) {
    trip(std::integral_constant<int, 0>{}, j, sa, sb);
    if (j + 1 < n_tiles) trip(std::integral_constant<int, 1>{}, j + 1, sb, sa);
  }

  const float l_tot = l_run + __shfl_xor(l_run, 32);
  const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
  {
    // Output through LDS (the K / V rings are idle: the last trip ended with a barrier): a lane holds 64 of its query's 128
    // values in 4-value pieces; each wave assembles its 32 rows x 256 bytes in a private region (chunk c of row r in
    // slot c ^ (r & 15)), reads whole 16-byte chunks back and stores full rows -- 8 stores of 16 bytes per lane instead
    // of 16 of 8 bytes that each touch 32 rows.
    char* ep = lds + wave * 8192;
    // (the lane id is taken afresh: addresses derived from the kernel's own `lane` are invariant over the passes of a
    // causal pair, get hoisted in front of the pass loop and then occupy registers all through the key walk)
    const int el = CAUSAL ? opaque_lane_id() : lane;
    const int e32 = el & 31, eh = el >> 5;
#pragma unroll
    for (int dt = 0; dt < 4; dt++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        half4 v = {cvt16<BF>(oacc[dt][4 * q] * inv), cvt16<BF>(oacc[dt][4 * q + 1] * inv), cvt16<BF>(oacc[dt][4 * q + 2] * inv),
                   cvt16<BF>(oacc[dt][4 * q + 3] * inv)};
        *reinterpret_cast<half4*>(ep + e32 * 256 + (((dt * 4 + q) ^ (e32 & 15)) * 16) + 8 * eh) = v;
      }
    const int er = el >> 4, ec = el & 15;
#pragma unroll
    for (int it = 0; it < 8; it++) {
      const int row = it * 4 + er;
      const half8 v = *reinterpret_cast<const half8*>(ep + row * 256 + ((ec ^ (row & 15)) * 16));
      if (wq0 + row < Sq) *reinterpret_cast<half8*>(Ob + (size_t)(wq0 + row) * lay.o_r + ec * 8) = v;
    }
    if (CAUSAL) __syncthreads();  // the next pass loads K / V tiles over these regions
  }
  }  // pass
}


// Packed sequences of different lengths (the VARLEN form of fa_fwd_d128_m16): the queries of sequence s are the rows
// [cu_q[s], cu_q[s + 1]) of one token stream, its keys and values the rows [cu_k[s], cu_k[s + 1]) of another.  The query heads that
// share a K/V head are packed: query row r of a (sequence, K/V head) is token r / group, head r % group, so that a block of
// 128 rows spans 128 / group tokens -- short sequences fill their blocks (a one-token sequence is one workgroup per K/V
// head) and less of a block's last tile is masked.
struct FaVarlen {
  const int *cu_q, *cu_k;  // [num_seqs + 1]
  int num_seqs, total_q, total_k;
  int group_shift;         // log2(group), -1 if the group is no power of two
  int zero_rest;           // also write zeros to the query rows in front of the first and behind the last sequence
  int pairs;               // (causal) a unit is a pair of query blocks, else one block
  int ranked;              // hand out the units of the sequence with the most keys first (up to 64 sequences)
  int chunks;              // a block's keys are cut into up to so many chunks, a workgroup each (1: they are not)
  float *part_acc, *part_ml;  // (chunks > 1) [total_q][query heads][chunks][128], [..][2]
};

// How the key tiles of one block of query rows are cut: `count` chunks of `tiles` each (the last may have fewer), none
// shorter than FA_MIN_CHUNK but by that.  The workgroups and the kernel that joins their results agree on it.
constexpr int FA_MIN_CHUNK = 4, FA_MAX_CHUNKS = 16;
struct FaChunks { int count, tiles; };
__device__ __forceinline__ FaChunks fa_chunks(int n_tiles, int most) {
  int c = (n_tiles + FA_MIN_CHUNK - 1) / FA_MIN_CHUNK;
  c = c < 1 ? 1 : (c > most ? most : c);
  FaChunks ch;
  ch.tiles = (n_tiles + c - 1) / c;
  ch.count = n_tiles > 0 ? (n_tiles + ch.tiles - 1) / ch.tiles : 1;
  return ch;
}

// Rows [begin, begin + len) of sequence s; offsets outside the stream are cut to it, a negative length counts as 0.
__device__ __forceinline__ int fa_seq_range(const int* cu, int s, int total, int& begin) {
  int b = cu[s], e = cu[s + 1];
  b = b < 0 ? 0 : (b > total ? total : b);
  e = e < b ? b : (e > total ? total : e);
  begin = b;
  return e - b;
}

// A unit's place: what the workgroup with place `loc` works on when every unit takes `per_unit` places (K/V heads).
struct FaUnit {
  int q_first, q_len, k_first, k_len;  // the sequence's rows
  int inside, units;                   // place among the sequence's, and how many units those are per K/V head
};

// Finds it; false behind the last unit.  Every wave by itself, one sequence per lane and 64 at a time: in order of falling
// key length (ranked), so that short sequences make up the tail of the grid, or as they come.
__device__ __forceinline__ bool fa_find_unit(const FaVarlen& vl, int group, int block_rows, int per_unit, int loc, FaUnit& u) {
  const int lane = threadIdx.x & 63, at = loc / per_unit;
  int base = 0;
  for (int s0 = 0; s0 < vl.num_seqs; s0 += 64) {
    int qf = 0, ql = 0, kf = 0, kl = -1, n = 0, before = 0;
    if (s0 + lane < vl.num_seqs) {
      ql = fa_seq_range(vl.cu_q, s0 + lane, vl.total_q, qf);
      kl = fa_seq_range(vl.cu_k, s0 + lane, vl.total_k, kf);
      n = (ql * group + block_rows - 1) / block_rows;
      if (vl.pairs) n = (n + 1) >> 1;
    }
    if (vl.ranked) {
      // one number per sequence orders them: more keys first, then as they come; lanes behind the last have no units
      const int key = kl < 0 ? -1 : (kl << 6) | (63 - lane);
      for (int j0 = 0; j0 < vl.num_seqs; j0 += 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int kj = __builtin_amdgcn_readlane(key, j0 + e), nj = __builtin_amdgcn_readlane(n, j0 + e);
          before += kj > key ? nj : 0;
        }
      }
    } else {
      int incl = n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(incl, d);
        if (lane >= d) incl += up;
      }
      before = base + incl - n;
      base += __builtin_amdgcn_readlane(incl, 63);
    }
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(before <= at && at < before + n);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      u.q_first = __builtin_amdgcn_readlane(qf, l), u.q_len = __builtin_amdgcn_readlane(ql, l);
      u.k_first = __builtin_amdgcn_readlane(kf, l), u.k_len = __builtin_amdgcn_readlane(kl, l);
      u.units = __builtin_amdgcn_readlane(n, l);
      u.inside = loc - __builtin_amdgcn_readlane(before, l) * per_unit;
      return true;
    }
  }
  return false;
}

// Drafted token trees over a paged cache (the TREE form of fa_fwd_d128_m16): the query rows of a (sequence, kv head) are all its
// nodes' heads, row r = node r / group, head r % group; see paged_tree.hip for the operator.
struct FaTree : FaPaged {
  const int* parents;           // [batch][nodes]
  float *part_acc, *part_ml;    // [batch][nodes][query heads][splits][128], [..][2]
  int nodes, num_kv_heads, num_seqs, row_blocks, num_splits;
  unsigned per_half;
};

// Measured, causal, the packed forms: 32 prompts of 1 to 300 tokens (32 query heads over 8) 26 us (744 workgroups of 1 to 5 tiles
// on 512 places; a single prompt of 16 tokens takes 6.6, an empty launch 3.6); 12 of 100 to 700 tokens behind up to 1500 (16 heads
// over one) 40 us, bound by LDS reads: the waves of a 64-row block split its rows and read every tile whole, 0.85 us a tile, the
// longest blocks 31 of them; 4 of 1500 to 8192 1.08 to 1.13 ms, 1.0 to 1.05 PFLOP/s, the rate of the rectangular form.
// Weights enter the second product in 16 bits; the sum that normalises them is that of the rounded ones.
enum class FaForm { PLAIN, PAGED, VARLEN, CHUNKED, TREE };  // CHUNKED: VARLEN with keys cut into chunks
template <FaForm F>
using FaFormArgs = std::conditional_t<F == FaForm::VARLEN || F == FaForm::CHUNKED, FaVarlen, std::conditional_t<F == FaForm::TREE, FaTree, FaPaged>>;

// The pipelined form on v_mfma_f32_16x16x32 (variant "..._m16").  Same tiles, rings, loads, passes and barriers as
// fa_fwd_d128_pipe; what changes is the MFMA shape and with it every fragment layout.  On benchmark-like data a
// 16x16x32 MFMA costs the board less energy per flop than a 32x32x16 (register-only loops with this tile's structure:
// 0.75 against 0.66 of the datasheet peak for the MFMAs alone, 0.60 against 0.57 with the softmax), and the prefill
// kernel runs against the power limit.
// A wave's 32 queries are two groups of 16 (qg), a 64-key tile four groups of 16 keys (kg), d = 128 four steps of 32 (ks),
// eight groups of 16 (dg).  With q16 = lane & 15, g = lane >> 4:
//   S^T(kg, qg) = K(kg) . Q(qg)^T:  A = K rows kg*16 + q16, d = 32 ks + 8 g .. + 7 (one 16-byte chunk from LDS, shared by
//       both query groups); B = Q row qg*16 + q16, same d (registers); the lane receives keys kg*16 + 4 g + r, r < 4, of
//       query qg*16 + q16: it owns one query per group and a quarter of the tile's keys.
//   O^T(dg, qg) += V(dg)^T . P(qg)^T over two steps of 32 keys (key groups 2 st, 2 st + 1): the lane's eight probabilities
//       (4 of either key group) are the B operand as they stand; A = V^T rows d = dg*16 + q16 for those same keys: two
//       transpose reads, each a 4 x 16 block (keys 4 g .. 4 g + 3 of one key group, 16 consecutive d) per 16 lanes.
// LDS: K chunk c of row r in slot c ^ (r & 15) as before; V chunk c of row r in slot c ^ 2 (r & 7): the 8 rows a half
// wave's transpose read touches (32 bytes each) then fall on 8 distinct 32-byte bank groups.
// SPREAD: the exponentials of a tile's second key step run behind the first key step's output MFMAs instead of behind
// the score MFMAs (vector work behind 48 of the trip's 64 MFMAs instead of 32).  Measured on 2 x 32 x 4096: ahead with
// eight waves (unmasked 475 against 484 us), behind with four (causal 268 against 263); each form is built the way it
// runs faster.
// QG: groups of 16 query rows per wave, 2 but for packed and tree calls with few rows.
template <bool CAUSAL, bool BF, int NW, bool SPREAD, FaForm FORM = FaForm::PLAIN, int QG = 2>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fa_fwd_d128_m16(
    const half_t* __restrict__ Q, const half_t* __restrict__ K, const half_t* __restrict__ V, half_t* __restrict__ O, int BH,
    int Sq_arg, int Sk_arg, float scale_log2e, int q_blocks_arg, FaLayout lay, FaFormArgs<FORM> pg) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  constexpr bool VARLEN = FORM == FaForm::VARLEN || FORM == FaForm::CHUNKED, TREE = FORM == FaForm::TREE, PAGED = FORM == FaForm::PAGED || TREE;
  static_assert(NW == 4 || !PAGED, "the paged form maps one page to one wave-load of a 4-wave workgroup");
  static_assert(!TREE || !CAUSAL, "the tree form masks by ancestors");
  // EXACT: the query fragments are the operand's own bits and scores are scaled in 32 bits, one multiplication per score;
  // otherwise scale . log2(e) is folded into the query and rounded to 16 bits again.
  constexpr bool EXACT = VARLEN || TREE;
  // CLEAN: what a query does not see does not reach it, whatever it holds: a weight of zero times a non-finite V entry would
  // be NaN, so tiles with masked keys are looked over first (clean_v).  That costs 1 us of 26 for 32 short prompts, 0.6 % for
  // long ones and 3 % for trees of 64 rows.
  constexpr bool CLEAN = (VARLEN && CAUSAL) || TREE;
  // CHUNKS: the keys may be cut into chunks, each for a workgroup of its own.
  constexpr bool CHUNKS = TREE || FORM == FaForm::CHUNKED;
  constexpr int WAVE_M = QG * 16, BLOCK_M = NW * WAVE_M, NI = 16 / NW;
  constexpr int TILE_B = FA_BLOCK_N * 256, VBUF = 2 * TILE_B;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q16 = lane & 15, g = lane >> 4;

  int Sq = Sq_arg, Sk = Sk_arg, q_blocks = q_blocks_arg;
  int units = CAUSAL ? (q_blocks + 1) / 2 : q_blocks;
  int bh, unit, b_idx, h_idx;
  size_t q_first = 0, k_first = 0;  // (VARLEN) the sequence's first rows
  int seq_q = 0;                    // (VARLEN) its query tokens; Sq counts rows
  int split = 0, first_tile = 0;    // (CHUNKS) the chunk of the keys, and where it begins
  int chunk_tiles = 0;              // (TREE) tiles of a chunk
  if constexpr (VARLEN) {
    const int pid = blockIdx.x;
    if (pg.zero_rest) {
      int first, last;
      fa_seq_range(pg.cu_q, 0, pg.total_q, first);
      const int len = fa_seq_range(pg.cu_q, pg.num_seqs - 1, pg.total_q, last);
      last += len;
      const long long outside = (long long)(first + pg.total_q - last) * lay.H;  // head rows, sixteen lanes each
      for (long long i = (long long)pid * (NW * 4) + (threadIdx.x >> 4); i < outside; i += (long long)gridDim.x * (NW * 4)) {
        const int r = (int)(i / lay.H), hd = (int)(i - (long long)r * lay.H);
        half_t* row = O + (size_t)(r < first ? r : last + r - first) * lay.o_r + hd * lay.o_h;
        *reinterpret_cast<half8*>(row + q16 * 8) = half8{};
      }
    }
    // A K/V head's units sit on one XCD when the K/V heads divide over the eight.
    const int kv_heads = lay.H / lay.group;
    const bool spread = kv_heads % 8 == 0;
    FaUnit u;
    int per_unit = spread ? kv_heads / 8 : kv_heads;
    if constexpr (CHUNKS) per_unit *= pg.chunks;
    if (!fa_find_unit(pg, lay.group, BLOCK_M, per_unit, spread ? pid >> 3 : pid, u)) return;
    units = u.units;
    int kv = u.inside / units;
    unit = u.inside - kv * units;
    if constexpr (CHUNKS) {
      split = kv % pg.chunks;
      kv /= pg.chunks;
    }
    h_idx = (spread ? kv * 8 + (pid & 7) : kv) * lay.group;
    q_first = u.q_first, k_first = u.k_first;
    Sq = u.q_len * lay.group;
    Sk = u.k_len;
    seq_q = u.q_len;
    q_blocks = (Sq + BLOCK_M - 1) / BLOCK_M;
    bh = b_idx = 0;
  } else if constexpr (TREE) {
    // kv heads next to each other (they read the same pages), then row blocks, then pieces of work
    int pid = blockIdx.x;
    const int kvh = pid % pg.num_kv_heads;
    pid /= pg.num_kv_heads;
    unit = pid % pg.row_blocks;
    const int reach = (pg.max_pages * 16) << pg.page_shift, chunk_steps = tree_chunk_steps(pg.seq_lens, pg.num_seqs, pg.num_splits, pg.per_half, reach);
    if (!tree_item(pg.seq_lens, pg.num_seqs, pg.num_splits, chunk_steps, reach, pid / pg.row_blocks, b_idx, split)) return;
    chunk_tiles = chunk_steps / 2;
    h_idx = kvh * lay.group;
    bh = 0;
    Sq = pg.nodes * lay.group;
    q_blocks = units = pg.row_blocks;
  } else {
    const int pid = blockIdx.x;
    if (((BH / lay.group) & 7) == 0) {
      const int xcd = pid & 7, loc = pid >> 3, per_kv = units * lay.group;
      const int w = loc % per_kv;
      bh = ((loc / per_kv) * 8 + xcd) * lay.group + w / units;
      unit = w % units;
    } else {
      bh = pid / units;
      unit = pid % units;
    }
    b_idx = bh / lay.H;
    h_idx = bh - b_idx * lay.H;
  }
  const int hk_idx = h_idx / lay.group;
  if constexpr (PAGED) {
    // Sequences differ in length and workgroups are dispatched in grid order: take the sequences longest first,
    // so that the short ones make up the tail.  Thread t counts the sequences that come before sequence t.
    const int num_seqs = TREE ? 1 : BH / lay.H;
    if (num_seqs > 1 && num_seqs <= 256) {
      int* pick = reinterpret_cast<int*>(lds);
      const int t = threadIdx.x;
      if (t < num_seqs) {
        const int mine = pg.seq_lens[t];
        int rank = 0;
        for (int j = 0; j < num_seqs; j++) {
          const int other = pg.seq_lens[j];
          rank += (other > mine) || (other == mine && j < t);
        }
        if (rank == b_idx) *pick = t;
      }
      __syncthreads();
      b_idx = __builtin_amdgcn_readfirstlane(*pick);
      __syncthreads();  // the slot is part of the K ring
    }
    Sk = __builtin_amdgcn_readfirstlane(pg.seq_lens[b_idx]);
    const int cap = (pg.max_pages * 16) << pg.page_shift;
    Sk = Sk < 0 ? 0 : (Sk > cap ? cap : Sk);
  }
  bool single = true;  // (CHUNKS) there is one chunk only
  int draft0 = 0;      // (TREE) position of node 0
  if constexpr (TREE) {
    draft0 = Sk - pg.nodes;
    const int tiles = (Sk + FA_BLOCK_N - 1) / FA_BLOCK_N;
    first_tile = split * chunk_tiles;
    if (first_tile >= tiles && split > 0) return;  // chunk 0 of an empty sequence writes its zeros
    single = tiles <= chunk_tiles;
    // the ancestors of this block's rows, behind the rings
    unsigned long long* seen = reinterpret_cast<unsigned long long*>(lds + 2 * FA_STAGE);
    if (wave == 0) seen[lane] = tree_ancestors(pg.parents + (size_t)b_idx * pg.nodes, pg.nodes);
    __syncthreads();
    unsigned long long mine = 0;
    if (threadIdx.x < BLOCK_M && unit * BLOCK_M + (int)threadIdx.x < Sq) mine = seen[(unit * BLOCK_M + threadIdx.x) / lay.group];
    __syncthreads();
    if (threadIdx.x < BLOCK_M) seen[threadIdx.x] = mine;
    __syncthreads();
  }
  // (VARLEN, TREE) the token, or node, of a packed query row, and where the row lies behind Qb (and Ob), in elements
  auto token_of = [&](int r) -> int {
    if constexpr (VARLEN) return pg.group_shift >= 0 ? r >> pg.group_shift : r / lay.group;
    else if constexpr (TREE) return r / lay.group;
    else return r;
  };
  auto row_at = [&](int r, unsigned pitch, int64_t head_pitch) -> size_t {
    if constexpr (VARLEN || TREE) {
      const int tok = token_of(r);
      return (size_t)tok * pitch + (size_t)(r - tok * lay.group) * head_pitch;
    } else {
      return (size_t)r * pitch;
    }
  };
  const int causal_off = Sk - (VARLEN ? seq_q : Sq);
  const half_t* Qb = Q + (VARLEN ? q_first * lay.q_r : b_idx * lay.q_b) + h_idx * lay.q_h;
  const half_t* Kb = K + (PAGED ? 0 : VARLEN ? k_first * lay.k_r : b_idx * lay.k_b) + hk_idx * lay.k_h;
  const half_t* Vb = V + (PAGED ? 0 : VARLEN ? k_first * lay.v_r : b_idx * lay.v_b) + hk_idx * lay.v_h;
  half_t* Ob = O + (VARLEN ? q_first * lay.o_r : b_idx * lay.o_b) + h_idx * lay.o_h;

  // fragment read addresses, opaque (see fa_fwd_d128_pipe): K by step over d, V by d group
  typedef const __attribute__((address_space(3))) half8* lds_half8_t;
  unsigned k_frag[4], v_frag[8];
  {
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
      k_frag[ks] = (unsigned)(uintptr_t)MI355_LDS(char, lds + q16 * 256 + (((ks * 4 + g) ^ q16) * 16));
      asm volatile("" : "+v"(k_frag[ks]));
    }
    // lane i of a 16-lane group hands in row i / 4, halfs 4 (i % 4) .. + 3 of the 4 x 16 block
    const int row = 4 * g + (q16 >> 2), rr = row & 7;
    const int vb0 = VBUF + row * 256 + (rr << 5) + 16 * ((q16 & 3) >> 1) + 8 * (q16 & 1);
#pragma unroll
    for (int dg = 0; dg < 8; dg++) {
      v_frag[dg] = (unsigned)(uintptr_t)MI355_LDS(char, lds + (vb0 ^ (dg << 5)));
      asm volatile("" : "+v"(v_frag[dg]));
    }
  }

  int passes = CAUSAL ? 2 : 1;
  if constexpr (VARLEN) passes = pg.pairs ? 2 : 1;
  int* v_flag = reinterpret_cast<int*>(lds + 2 * FA_STAGE + (TREE ? BLOCK_M * 8 : 0));  // (CLEAN) a wave found one
  if constexpr (CLEAN) {
    if (threadIdx.x == 0) *v_flag = 0;
    __syncthreads();
  }
  for (int pass = 0; pass < passes; pass++) {
  const int qb = CAUSAL ? (pass == 0 ? q_blocks - 1 - unit : unit) : unit;
  if (CAUSAL && pass == 1 && 2 * unit == q_blocks - 1) break;
  const int q0 = qb * BLOCK_M;
  const int wq0 = q0 + wave * WAVE_M;
  const int wave_first = token_of(wq0), wave_last = token_of(wq0 + WAVE_M - 1);  // the wave's tokens

  int k_end = Sk;
  if (CAUSAL) {
    int last_q = q0 + BLOCK_M - 1;
    if (last_q > Sq - 1) last_q = Sq - 1;
    int lim = token_of(last_q) + causal_off + 1;
    if (lim < k_end) k_end = lim;
  }
  int n_tiles = k_end > 0 ? (k_end + FA_BLOCK_N - 1) / FA_BLOCK_N : 0;
  if constexpr (TREE) {
    n_tiles -= first_tile;
    n_tiles = n_tiles < chunk_tiles ? n_tiles : chunk_tiles;
  } else if constexpr (CHUNKS) {
    const FaChunks ch = fa_chunks(n_tiles, pg.chunks);
    if (split >= ch.count) return;
    single = ch.count == 1;
    first_tile = split * ch.tiles;
    n_tiles -= first_tile;
    n_tiles = n_tiles < ch.tiles ? n_tiles : ch.tiles;
  }

  // Q fragments [query group][step over d], scale . log2(e) folded in and rounded to the 16-bit format again
  half8 qf[QG][4];
#pragma unroll
  for (int qg = 0; qg < QG; qg++) {
    const int q_row = wq0 + qg * 16 + q16;
#pragma unroll
    for (int ks = 0; ks < 4; ks++) {
      if (q_row < Sq) {
        const half8 raw = *reinterpret_cast<const half8*>(Qb + row_at(q_row, lay.q_r, lay.q_h) + ks * 32 + g * 8);
        if constexpr (EXACT) {
          qf[qg][ks] = raw;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) qf[qg][ks][e] = cvt16<BF>(to_f32<BF>(raw[e]) * scale_log2e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) qf[qg][ks][e] = (half_t)0;
      }
    }
  }

  const int lrow = lane >> 4, lslot = lane & 15;
  const int k_chunk = lslot ^ ((wave * 4 + lrow) & 15);
  const int v_chunk = lslot ^ (2 * (((wave & 1) << 2) | lrow));
  const unsigned k_rb = lay.k_r * 2, v_rb = lay.v_r * 2;
  const unsigned k_voff = (wave * 4 + lrow) * k_rb + k_chunk * 16;
  const unsigned v_voff = (wave * 4 + lrow) * v_rb + v_chunk * 16;
  // paged form: page ids come through the scalar cache (constant address space: the table is not written while the
  // kernel runs), one tile ahead of their use, so that no K/V load waits for a table read
  typedef const int __attribute__((address_space(4)))* table_ptr_t;
  table_ptr_t table_row = (table_ptr_t)0;
  if constexpr (PAGED) table_row = (table_ptr_t)(unsigned long long)(pg.block_table + (size_t)b_idx * pg.max_pages);
  auto load_ids = [&](int tile, int* ids) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int blk = tile * 4 + i, page = blk >> pg.page_shift;  // 16-token block -> its page and place in it
        const int e = page < pg.max_pages ? table_row[page] : -1;
        ids[i] = (e >= 0 && e < pg.num_pages) ? (e << pg.page_shift) + (blk & ((1 << pg.page_shift) - 1)) : -1;
      }
    }
  };
  auto issue_kv = [&](const half_t* base, unsigned rb, unsigned voff, int tile, int lds_off, const int* ids) {
    char* dst = lds + lds_off + wave * 1024;
    const int row0 = tile * FA_BLOCK_N;
    int rem = Sk - row0;
    rem = rem > FA_BLOCK_N ? FA_BLOCK_N : rem;
    if constexpr (PAGED) {
      // wave-load i covers rows 16 i .. 16 i + 15 of the tile = 16-token block 4 tile + i of the sequence: one descriptor
      // per block, sized to its valid rows (none for a block beyond the sequence or an id outside the cache)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int id = ids[i];
        int rows = rem - 16 * i;
        rows = rows > 16 ? 16 : rows;
        const bool ok = rows > 0 && id >= 0;
        const buffer_rsrc_t rs = make_buffer(reinterpret_cast<const char*>(base) + (size_t)(ok ? id : 0) * 16u * rb,
                                             ok ? (unsigned)(rows - 1) * rb + 256u : 0u);
        buffer_load_lds_16B(rs, voff, 0, dst + i * 4096);
      }
    } else {
      const buffer_rsrc_t rs = make_buffer(reinterpret_cast<const char*>(base) + (size_t)row0 * rb, (unsigned)(rem - 1) * rb + 256u);
#pragma unroll
      for (int i = 0; i < NI; i++) {
#if !defined(MI355_ABLATE_NO_LOADS)
        buffer_load_lds_16B(rs, voff + (unsigned)(i * NW * 4) * rb, 0, dst + i * NW * 1024);
#endif
      }
    }
  };

  // the j-th key tile that this workgroup walks
  auto tile_at = [&](int j) -> int {
    if constexpr (CHUNKS) return first_tile + j;
    else return j;
  };
  floatx4 oacc[8][QG];  // [d group][query group]
#pragma unroll
  for (int dg = 0; dg < 8; dg++)
#pragma unroll
    for (int qg = 0; qg < QG; qg++) oacc[dg][qg] = floatx4{0.f, 0.f, 0.f, 0.f};
  // the negated running maximum of the lane's query in either group, four equal values: the addend of every score chain
  floatx4 negm[QG] = {};
  float l_run[QG] = {};
  float grow_thr[QG];
  grow_thr[0] = grow_thr[QG - 1] = -INFINITY;
  const float score_mul = EXACT ? scale_log2e : 1.f;                // score units -> log2 units
  const float kRescaleThreshold = EXACT ? 8.f / scale_log2e : 8.f;  // 2^8, in score units

  auto wave_active = [&](int tile) {
    if constexpr (TREE) return wq0 < Sq;  // a wave without rows only loads
    else return !CAUSAL || (tile * FA_BLOCK_N <= wave_last + causal_off);
  };
  auto kread = [&](int f, int koff) {  // K fragment f = kg * 4 + ks of the slot at koff
#if defined(MI355_ABLATE_NO_K_READS)
    half8 stale = qf[0][f & 3];
    asm volatile("" : "+v"(stale));
    return stale;
#else
    return *(lds_half8_t)(uintptr_t)(k_frag[f & 3] + (unsigned)(koff + (f >> 2) * 4096));
#endif
  };
  // S^T of one tile, no softmax beside it (a pass's first tile)
  auto scores = [&](int koff, floatx4 (*s)[QG]) {
#pragma unroll
    for (int f = 0; f < 16; f++) {
      const int kg = f >> 2, ks = f & 3;
      const half8 kf = kread(f, koff);
#pragma unroll
      for (int qg = 0; qg < QG; qg++) s[kg][qg] = mfma16_16x16x32<BF>(kf, qf[qg][ks], ks == 0 ? negm[qg] : s[kg][qg]);
    }
  };

  // (CLEAN) Looks a masked tile's V over, a quarter per wave, and lets the waves know of a non-finite entry.  With none (one
  // barrier and 16 words per lane later) that is all.  Otherwise the entries are added by themselves to the queries that see
  // them -- infinity or NaN is what those sums become, whatever the weight -- and cleared in LDS.
  auto clean_v = [&](int tile, char* vt) {
    auto marks = [&](unsigned two) { return tree_nonfinite2<BF>(two); };
    uint4* mine = reinterpret_cast<uint4*>(vt) + threadIdx.x;
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < TILE_B / 16 / (NW * 64); i++) {
      const uint4 x = mine[i * NW * 64];
      any |= marks(x.x) | marks(x.y) | marks(x.z) | marks(x.w);
    }
    if (__builtin_amdgcn_ballot_w64(any != 0) != 0 && lane == 0) *v_flag = 1;
    // (not __syncthreads, which would wait for the tiles under way)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (*(volatile int*)v_flag == 0) return;
    const int key0 = tile * FA_BLOCK_N;
    unsigned long long set[QG];
    int lim[QG];
#pragma unroll
    for (int qg = 0; qg < QG; qg++) {
      if constexpr (TREE) set[qg] = reinterpret_cast<const unsigned long long*>(lds + 2 * FA_STAGE)[wave * WAVE_M + qg * 16 + q16];
      else lim[qg] = token_of(wq0 + qg * 16 + q16) + causal_off;
    }
#pragma unroll 1
    for (int j = 0; j < FA_BLOCK_N; j++) {
      unsigned sees[QG];  // all ones or zero
#pragma unroll
      for (int qg = 0; qg < QG; qg++) {
        if constexpr (TREE) sees[qg] = 0u - (tree_visible4(set[qg], key0 + j - draft0) & 1u);
        else sees[qg] = key0 + j <= lim[qg] ? ~0u : 0u;
      }
      const char* row = vt + j * 256 + (g & 1) * 8;
#pragma unroll
      for (int dg = 0; dg < 8; dg++) {
        const uint2 v = *reinterpret_cast<const uint2*>(row + (((2 * dg + (g >> 1)) ^ (2 * (j & 7))) * 16));
        const unsigned lo = v.x & (marks(v.x) >> 15) * 0xFFFFu, hi = v.y & (marks(v.y) >> 15) * 0xFFFFu;
#pragma unroll
        for (int qg = 0; qg < QG; qg++) {
          const unsigned a = lo & sees[qg], b = hi & sees[qg];
          const floatx4 add = {tree_value<BF>(a & 0xFFFFu), tree_value<BF>(a >> 16), tree_value<BF>(b & 0xFFFFu), tree_value<BF>(b >> 16)};
          oacc[dg][qg] = oacc[dg][qg] + add;
        }
      }
    }
    __syncthreads();
    auto clear = [&](unsigned two) {
      const unsigned b = marks(two) >> 15;
      return two & ~(b * 0xFFFFu);
    };
    for (int i = 0; i < TILE_B / 16 / (NW * 64); i++) {
      uint4 x = mine[i * NW * 64];
      x.x = clear(x.x), x.y = clear(x.y), x.z = clear(x.z), x.w = clear(x.w);
      mine[i * NW * 64] = x;
    }
    if (threadIdx.x == 0) *v_flag = 0;
    __syncthreads();
  };

  // `dropped` (TREE): bit i: the tile's 16-token block i has no page in the cache
  auto softmax_pv = [&](int tile, int dropped, auto voff_tag, floatx4 (*s)[QG], int koff_next, floatx4 (*s_next)[QG]) {
    constexpr int VOFF = decltype(voff_tag)::value;
    {
      const int key0 = tile * FA_BLOCK_N;
      if constexpr (TREE) {
        if (key0 + FA_BLOCK_N > draft0 || dropped) {
          const unsigned long long* seen = reinterpret_cast<const unsigned long long*>(lds + 2 * FA_STAGE) + wave * WAVE_M + q16;
#pragma unroll
          for (int qg = 0; qg < QG; qg++) {
            const unsigned long long set = seen[qg * 16];
#pragma unroll
            for (int kg = 0; kg < 4; kg++) {
              const unsigned vis = (dropped >> kg) & 1 ? 0u : tree_visible4(set, key0 + 16 * kg + 4 * g - draft0);
#pragma unroll
              for (int r = 0; r < 4; r++) s[kg][qg][r] = tree_hide(s[kg][qg][r], vis, r);
            }
          }
        }
      } else {
      const bool need_mask = (CAUSAL && (key0 + FA_BLOCK_N - 1 > wave_first + causal_off)) || (key0 + FA_BLOCK_N > Sk);
      if (need_mask) {
#pragma unroll
        for (int qg = 0; qg < QG; qg++) {
          const int q_row = wq0 + qg * 16 + q16;
          const int q_tok = token_of(q_row);
          const int lim = CAUSAL ? (q_tok + causal_off < Sk - 1 ? q_tok + causal_off : Sk - 1) : Sk - 1;  // last visible key
          const int rel = lim - key0 - 4 * g;
#pragma unroll
          for (int kg = 0; kg < 4; kg++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
              const unsigned hide = (unsigned)((rel - (16 * kg + r)) >> 31);
              const float sv = s[kg][qg][r];
              s[kg][qg][r] = __builtin_bit_cast(float, (hide & 0xFF800000u) | (~hide & __builtin_bit_cast(unsigned, sv)));
            }
        }
      }
      }
    }
    float mx[QG];
#pragma unroll
    for (int qg = 0; qg < QG; qg++) {
      mx[qg] = s[0][qg][0];
#pragma unroll
      for (int kg = 0; kg < 4; kg++)
#pragma unroll
        for (int r = 0; r < 4; r++) mx[qg] = fmaxf(mx[qg], s[kg][qg][r]);
    }
    if (__builtin_amdgcn_ballot_w64(mx[0] > grow_thr[0] || mx[QG - 1] > grow_thr[QG - 1]) != 0) {
      // rare: some query's scores outgrew its maximum (or it saw its first key).  A query's keys are spread over the
      // four lanes q16 + 16 g; they take the same decision.
#pragma unroll
      for (int qg = 0; qg < QG; qg++) {
        float mxx = fmaxf(mx[qg], __shfl_xor(mx[qg], 16));
        mxx = fmaxf(mxx, __shfl_xor(mxx, 32));
        if (mxx > grow_thr[qg]) {
          const bool fresh = grow_thr[qg] == -INFINITY;
          const float delta = fresh ? mxx : fmaxf(mxx, 0.f);  // (mxx > -inf here)
          const float alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(EXACT ? -delta * score_mul : -delta);
          grow_thr[qg] = kRescaleThreshold;
          l_run[qg] *= alpha;
#pragma unroll
          for (int dg = 0; dg < 8; dg++)
#pragma unroll
            for (int r = 0; r < 4; r++) oacc[dg][qg][r] *= alpha;
#pragma unroll
          for (int kg = 0; kg < 4; kg++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[kg][qg][r] -= delta;
#pragma unroll
          for (int r = 0; r < 4; r++) negm[qg][r] -= delta;
        }
      }
    }
    // Scores of the next tile and the softmax of this one, step by step.  Step i = MFMA (kg, ks, qg) = (i / 8, (i / 2) % 4,
    // i % 2) of the next tile -- a K fragment serves both query groups back to back and is requested three fragments
    // ahead -- and one exponential of this tile, taken in the order the output MFMAs want the probabilities: key step,
    // query group, key group of the pair, r.  Every second step packs a pair; its dot2 (the row sum of what the second
    // contraction multiplies) runs one pair behind.  The empty statements tie the vector work to its step.
    half8 pf[QG][2];  // [query group][key step]
    float psum[QG];
#pragma unroll
    for (int qg = 0; qg < QG; qg++) psum[qg] = 0.f;
    half2v pp_prev = {(half_t)0, (half_t)0};
    // exponential e of the tile (0..31), in the order the output MFMAs want the probabilities: key step e / 16, query group
    // (e / 8) % 2, key group of the pair (e / 4) % 2, r = e % 4.  Every second one packs a pair; the pair's dot2 (the row
    // sum of what the second contraction multiplies) runs one pair behind.  The empty statements tie the work to its step.
    float e_even = 0.f;
    auto expo = [&](int e) {
      const int st = e / (8 * QG), eq = (e >> 3) % QG, ekg = 2 * st + ((e >> 2) & 1), r = e & 3;
#if defined(MI355_ABLATE_NO_EXP)
      const float ev = s[ekg][eq][r];
#else
      const float ev = __builtin_amdgcn_exp2f(EXACT ? s[ekg][eq][r] * score_mul : s[ekg][eq][r]);
#endif
      if (e & 1) {
        if (e > 1) psum[((e - 2) >> 3) % QG] = dot2_ones<BF>(pp_prev, psum[((e - 2) >> 3) % QG]);
        half2v pp = cvt16x2<BF>(e_even, ev);
        if constexpr (QG == 2) asm volatile("" : "+v"(pp), "+v"(psum[0]), "+v"(psum[1]));
        else asm volatile("" : "+v"(pp), "+v"(psum[0]));
        pf[eq][st][((e >> 2) & 1) * 4 + r - 1] = pp[0];
        pf[eq][st][((e >> 2) & 1) * 4 + r] = pp[1];
        pp_prev = pp;
      } else {
        e_even = ev;
        asm volatile("" : "+v"(e_even));
      }
    };
    // Scores of the next tile, step by step: step i = MFMA (kg, ks, qg) = (i / 8, (i / 2) % 4, i % 2) -- a K fragment serves
    // both query groups back to back and is requested three fragments ahead -- with the exponentials of this tile's
    // FIRST key step behind every second MFMA; those of the second key step run behind the first key step's output
    // MFMAs below, so that the vector work is spread over 48 of the trip's 64 MFMAs.
    __builtin_amdgcn_sched_barrier(0);
    {
      half8 kf[4];
      kf[0] = kread(0, koff_next);
      kf[1] = kread(1, koff_next);
      kf[2] = kread(2, koff_next);
#pragma unroll
      for (int i = 0; i < 16 * QG; i++) {
        const int f = i / QG, kg = f >> 2, ks = f & 3, qg = i % QG;
        if (qg == 0 && f + 3 < 16) kf[(f + 3) & 3] = kread(f + 3, koff_next);
        s_next[kg][qg] = mfma16_16x16x32<BF>(kf[f & 3], qf[qg][ks], ks == 0 ? negm[qg] : s_next[kg][qg]);
        if (SPREAD) {
          if (i & 1) expo(i >> 1);
        } else {
          expo(i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // O^T += V^T P^T: step f = (key step, d group) = (f / 8, f % 8), two MFMAs (one per query group) on one V^T fragment
    // (two transpose reads, in assembly with their waits, see fa_fwd_d128_pipe), requested two fragments ahead.
    half4 vlo[3], vhi[3];
    auto vr = [&](auto ftag) {  // fragment f = st * 8 + dg
      constexpr int f = decltype(ftag)::value;
      constexpr int off = VOFF + (f >> 3) * 8192;  // key groups 2 st and 2 st + 1: 16 rows of 256 bytes apart
      half4 &lo = vlo[f % 3], &hi = vhi[f % 3];
      const unsigned addr = v_frag[f & 7];
#if defined(MI355_ABLATE_NO_V_READS)
      asm volatile("" : "=&v"(lo), "=&v"(hi) : "v"(addr));
#else
      asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                   : "=&v"(lo), "=&v"(hi)
                   : "v"(addr), "n"(off), "n"(off + 4096));
#endif
    };
    vr(std::integral_constant<int, 0>{});
    vr(std::integral_constant<int, 1>{});
    static_for<0, 16>([&](auto ftag) {
      constexpr int f = decltype(ftag)::value;
      constexpr int st = f >> 3, dg = f & 7;
      if constexpr (f + 2 < 16) vr(std::integral_constant<int, f + 2>{});
      half4 &lo = vlo[f % 3], &hi = vhi[f % 3];
      if constexpr (f + 2 < 16)
        asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(lo), "+v"(hi));
      else if constexpr (f + 1 < 16)
        asm volatile("s_waitcnt lgkmcnt(2)" : "+v"(lo), "+v"(hi));
      else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(lo), "+v"(hi));
      const half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      oacc[dg][0] = mfma16_16x16x32<BF>(vf, pf[0][st], oacc[dg][0]);
      if constexpr (SPREAD && f < 8) expo(16 + 2 * f);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (QG == 2) {
        oacc[dg][1] = mfma16_16x16x32<BF>(vf, pf[1][st], oacc[dg][1]);
        if constexpr (SPREAD && f < 8) expo(16 + 2 * f + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (f == 7 || (!SPREAD && f == 0)) {  // the last pair's dot2 (it belongs to query group 1)
        if (SPREAD || f == 0) {
          psum[QG - 1] = dot2_ones<BF>(pp_prev, psum[QG - 1]);
#pragma unroll
          for (int qg = 0; qg < QG; qg++) l_run[qg] += psum[qg];
        }
      }
    });
  };

  floatx4 sa[4][QG], sb[4][QG];  // scores [key group][query group], two tiles
  int k_ids[4] = {-1, -1, -1, -1}, v_ids[4] = {-1, -1, -1, -1};  // paged form: ids of the next K tile and the next V tile to fetch
  // (TREE) which blocks of the present tile, the next one and the one behind have no page.  The plain paged form lets their
  // rows read as zeros; a tree's query must not count them.
  int drop0 = 0, drop1 = 0, drop2 = 0;
  auto drops = [&](const int* ids) {
    int d = 0;
    if constexpr (TREE) {
#pragma unroll
      for (int i = 0; i < 4; i++) d |= (ids[i] < 0) << i;
    }
    return d;
  };
  if (n_tiles > 0) {
    load_ids(tile_at(0), k_ids);
    drop0 = drops(k_ids);
    issue_kv(Kb, k_rb, k_voff, tile_at(0), 0, k_ids);
    issue_kv(Vb, v_rb, v_voff, tile_at(0), VBUF, k_ids);
    load_ids(tile_at(1), v_ids);
    drop1 = drops(v_ids);
    if (n_tiles > 1) issue_kv(Kb, k_rb, k_voff, tile_at(1), TILE_B, v_ids);
    load_ids(tile_at(2), k_ids);  // what trip 0 issues: K(2) and V(1)
    drop2 = drops(k_ids);
    wait_vmcnt0();
    __syncthreads();
    if (wave_active(tile_at(0))) scores(0, sa);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
  }
  auto trip = [&](auto par_tag, int j, floatx4 (*s_cur)[QG], floatx4 (*s_next)[QG]) {
    constexpr int PAR = decltype(par_tag)::value;
    constexpr int K_CUR = PAR * TILE_B, K_NEXT = (1 - PAR) * TILE_B, V_CUR = VBUF + PAR * TILE_B, V_NEXT = VBUF + (1 - PAR) * TILE_B;
    if (j + 2 < n_tiles) issue_kv(Kb, k_rb, k_voff, tile_at(j + 2), K_CUR, k_ids);
    if (j + 1 < n_tiles) issue_kv(Vb, v_rb, v_voff, tile_at(j + 1), V_NEXT, v_ids);
    const int dropped = drop0;
    if constexpr (PAGED) {
      // the next trip fetches V(j+2) -- the tile whose ids K just used -- and K(j+3)
#pragma unroll
      for (int i = 0; i < 4; i++) v_ids[i] = k_ids[i];
      load_ids(tile_at(j + 3), k_ids);
      if constexpr (TREE) {
        drop0 = drop1;
        drop1 = drop2;
        drop2 = drops(k_ids);
      }
    }
    if constexpr (CLEAN) {
      // some query of the workgroup does not see some key of the tile
      const int first_hidden = TREE ? draft0 : token_of(q0) + causal_off + 1;
      if ((tile_at(j) + 1) * FA_BLOCK_N > first_hidden) clean_v(tile_at(j), lds + V_CUR);
    }
    if (wave_active(tile_at(j))) softmax_pv(tile_at(j), dropped, std::integral_constant<int, V_CUR - VBUF>{}, s_cur, K_NEXT, s_next);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#if !defined(MI355_ABLATE_NO_BARRIERS)
    __syncthreads();
#endif
  };
  for (int j = 0; j < n_tiles; j += 2) {
    trip(std::integral_constant<int, 0>{}, j, sa, sb);
    if (j + 1 < n_tiles) trip(std::integral_constant<int, 1>{}, j + 1, sb, sa);
  }

  if (CHUNKS && !single) {
    // partial results of the chunk: the unnormalised sums, their maximum in log2 units and weight
    if constexpr (CHUNKS) {
      const int el = opaque_lane_id(), e16 = el & 15, eg = el >> 4;
#pragma unroll
      for (int qg = 0; qg < QG; qg++) {
        float l_tot = l_run[qg] + __shfl_xor(l_run[qg], 16);
        l_tot += __shfl_xor(l_tot, 32);
        const int r = wq0 + qg * 16 + e16;
        if (r < Sq) {
          const int tok = token_of(r);  // or node
          size_t at;
          if constexpr (TREE) at = (((size_t)b_idx * pg.nodes + tok) * lay.H + h_idx + (r - tok * lay.group)) * pg.num_splits + split;
          else at = ((q_first + tok) * lay.H + h_idx + (r - tok * lay.group)) * pg.chunks + split;
          float* acc = pg.part_acc + at * 128 + 4 * eg;
#pragma unroll
          for (int dg = 0; dg < 8; dg++) *reinterpret_cast<floatx4*>(acc + dg * 16) = oacc[dg][qg];
          if (eg == 0) {
            pg.part_ml[at * 2] = grow_thr[qg] == -INFINITY ? -INFINITY : -negm[qg][0] * score_mul;
            pg.part_ml[at * 2 + 1] = l_tot;
          }
        }
      }
    }
  } else {
    // Output through LDS (the rings are idle: the last trip ended with a barrier): each wave assembles its 32 rows x 256
    // bytes in a private region (chunk c of row r in slot c ^ (r & 15)) from 8-byte pieces -- the lane holds d = 16 dg +
    // 4 g .. + 3 of its query in either group -- and stores whole rows, 16 bytes per lane.
    char* ep = lds + wave * 8192;
    const int el = (CAUSAL || EXACT) ? opaque_lane_id() : lane;  // (see fa_fwd_d128_pipe)
    const int e16 = el & 15, eg = el >> 4;
#pragma unroll
    for (int qg = 0; qg < QG; qg++) {
      float l_tot = l_run[qg] + __shfl_xor(l_run[qg], 16);
      l_tot += __shfl_xor(l_tot, 32);
      const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
#pragma unroll
      for (int dg = 0; dg < 8; dg++) {
        const half4 v = {cvt16<BF>(oacc[dg][qg][0] * inv), cvt16<BF>(oacc[dg][qg][1] * inv), cvt16<BF>(oacc[dg][qg][2] * inv),
                         cvt16<BF>(oacc[dg][qg][3] * inv)};
        *reinterpret_cast<half4*>(ep + (qg * 16 + e16) * 256 + (((dg * 2 + (eg >> 1)) ^ e16) * 16) + 8 * (eg & 1)) = v;
      }
    }
    const int er = el >> 4, ec = el & 15;
#pragma unroll
    for (int it = 0; it < WAVE_M / 4; it++) {
      const int row = it * 4 + er;
      const half8 v = *reinterpret_cast<const half8*>(ep + row * 256 + ((ec ^ (row & 15)) * 16));
      if (wq0 + row < Sq) *reinterpret_cast<half8*>(Ob + row_at(wq0 + row, lay.o_r, lay.o_h) + ec * 8) = v;
    }
    if (CAUSAL) __syncthreads();  // the next pass loads K / V tiles over these regions
  }
  }  // pass
}

// Joins the chunks of packed sequences' rows (up to 64 sequences): 32 lanes of 16 bytes per row, two rows per wave.  Rows of
// one chunk were written by the attention kernel, rows outside every sequence are left alone.
template <bool BF>
__global__ __launch_bounds__(256) void fa_varlen_join(FaVarlen vl, FaLayout lay, half_t* __restrict__ O, int causal) {
  const int lane = threadIdx.x & 63, l32 = lane & 31;
  const long long rows = (long long)vl.total_q * lay.H;
  const long long first = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * 2;  // the wave's rows: this one and the next
  int qf = 0, ql = 0, kf = 0, kl = 0;
  if (lane < vl.num_seqs) {
    ql = fa_seq_range(vl.cu_q, lane, vl.total_q, qf);
    kl = fa_seq_range(vl.cu_k, lane, vl.total_k, kf);
  }
  int seq = -1, tok = 0, head = 0;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const long long r = first + h < rows ? first + h : rows - 1;
    const int t = (int)(r / lay.H);
    const unsigned long long hit = __builtin_amdgcn_ballot_w64(qf <= t && t < qf + ql);
    if ((lane >> 5) == h) {
      seq = first + h < rows && hit ? __builtin_ctzll(hit) : -1;
      tok = t;
      head = (int)(r - (long long)t * lay.H);
    }
  }
  const int from = seq < 0 ? 0 : seq;
  const int q_first = __shfl(qf, from), q_len = __shfl(ql, from), k_len = __shfl(kl, from);
  if (seq < 0) return;
  // the row's block, its key tiles and their chunks, as in the attention kernel
  const int row = (tok - q_first) * lay.group + head % lay.group;
  int last = row / 64 * 64 + 63;
  last = last < q_len * lay.group ? last : q_len * lay.group - 1;
  int k_end = causal ? last / lay.group + (k_len - q_len) + 1 : k_len;
  k_end = k_end < k_len ? k_end : k_len;
  const int n = fa_chunks(k_end > 0 ? (k_end + FA_BLOCK_N - 1) / FA_BLOCK_N : 0, vl.chunks).count;
  if (n == 1) return;
  const size_t at = ((size_t)tok * lay.H + head) * vl.chunks;
  const float* ml = vl.part_ml + at * 2;
  const float* acc = vl.part_acc + at * 128 + l32 * 4;
  float m_tot = -INFINITY;
  for (int c = 0; c < n; c++) m_tot = fmaxf(m_tot, ml[2 * c]);
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int c = 0; c < n; c++) {
    // (no maximum: zeros, or a row of scores that are not numbers; either is passed on as it is)
    const float w = m_tot > -INFINITY ? __builtin_amdgcn_exp2f(ml[2 * c] - m_tot) : 1.f;
    const floatx4 p = *reinterpret_cast<const floatx4*>(acc + (size_t)c * 128);
    l = __builtin_fmaf(w, ml[2 * c + 1], l);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(w, p[e], o[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const half4 v = {cvt16<BF>(o[0] * inv), cvt16<BF>(o[1] * inv), cvt16<BF>(o[2] * inv), cvt16<BF>(o[3] * inv)};
  *reinterpret_cast<half4*>(O + (size_t)tok * lay.o_r + (size_t)head * lay.o_h + l32 * 4) = v;
}

// Persistent form of fa_fwd_d128_pipe ("walk"): one workgroup per CU slot runs its passes (a pass = one block of
// NW * 32 queries of one head against its keys) one after the other -- units dealt round-robin (unit = workgroup +
// i * grid), a causal unit being a pair of blocks as above -- and overlaps what a pass costs beside its key tiles:
//  * the next pass's Q rows and first tiles (K 0, K 1, V 0) are requested in front of the current pass's LAST tile when
//    that tile has odd number (a pass of an even tile count): both K slots and V slot 0 are free from there on, the Q
//    rows land in registers that would hold the scores of a following tile (the last tile computes none), and nothing
//    waits for any of it before the finished pass has been normalised and staged.  Otherwise they are requested right
//    after the last trip;
//  * the output goes through a staging region of its own (the rings are being filled) and is stored behind the barrier
//    that opens the next pass; the stores are not waited for: they drain under the next pass's first trip, whose
//    closing wait covers them.
// A pass has at least two key tiles (the launcher checks Sk >= 128, and Sq == Sk with the mask).  The arithmetic per
// query is that of fa_fwd_d128_pipe, instruction for instruction: results are bit-identical.
template <bool CAUSAL, bool BF, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fa_fwd_d128_walk(
    const half_t* __restrict__ Q, const half_t* __restrict__ K, const half_t* __restrict__ V, half_t* __restrict__ O, int BH,
    int Sq, int Sk, float scale_log2e, int q_blocks, FaLayout lay) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  constexpr int BLOCK_M = NW * 32, NI = 16 / NW;
  constexpr int TILE_B = FA_BLOCK_N * 256, VBUF = 2 * TILE_B, STG = 4 * TILE_B;  // K ring, V ring, output staging
  constexpr int STG_ROWS = NW == 8 ? 32 : 8;  // rows a wave stages per round: 8 KiB (one round) or 2 KiB (four) per wave
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  const int causal_off = Sk - Sq;
  const int units = CAUSAL ? (q_blocks + 1) / 2 : q_blocks;
  const int total_units = BH * units;
  const bool xcd_map = ((BH / lay.group) & 7) == 0;  // the launcher makes the grid a multiple of 8 then

  // ---- passes of this workgroup, by ordinal: unit = blockIdx.x + (ord / passes per unit) * gridDim.x ----
  struct Pass {
    int ord;  // < 0: there is no such pass
    int b, hq, hk, qb, n;  // batch, query head, K/V head, query block, key tiles
  };
  auto pass_at = [&](int ord) {  // the first existing pass with ordinal >= ord
    Pass ps;
    for (;;) {
      const int pid = (int)blockIdx.x + (CAUSAL ? (ord >> 1) : ord) * (int)gridDim.x;
      if (pid >= total_units) {
        ps.ord = -1, ps.b = ps.hq = ps.hk = ps.qb = 0, ps.n = 2;
        return ps;
      }
      int bh, unit;
      if (xcd_map) {
        const int xcd = pid & 7, loc = pid >> 3, per_kv = units * lay.group;
        const int w = loc % per_kv;
        bh = ((loc / per_kv) * 8 + xcd) * lay.group + w / units;
        unit = w % units;
      } else {
        bh = pid / units;
        unit = pid % units;
      }
      const bool second = CAUSAL && (ord & 1);
      if (second && 2 * unit == q_blocks - 1) {  // the middle block of an odd count has no partner
        ord++;
        continue;
      }
      ps.ord = ord;
      ps.qb = CAUSAL ? (second ? unit : q_blocks - 1 - unit) : unit;
      ps.b = bh / lay.H;
      ps.hq = bh - ps.b * lay.H;
      ps.hk = ps.hq / lay.group;
      int k_end = Sk;
      if (CAUSAL) {
        int last_q = ps.qb * BLOCK_M + BLOCK_M - 1;
        if (last_q > Sq - 1) last_q = Sq - 1;
        const int lim = last_q + causal_off + 1;
        if (lim < k_end) k_end = lim;
      }
      ps.n = (k_end + FA_BLOCK_N - 1) / FA_BLOCK_N;
      // (the divisions run on the vector unit; the fields are wave-uniform and belong in scalar registers)
      ps.qb = __builtin_amdgcn_readfirstlane(ps.qb), ps.b = __builtin_amdgcn_readfirstlane(ps.b);
      ps.hq = __builtin_amdgcn_readfirstlane(ps.hq), ps.hk = __builtin_amdgcn_readfirstlane(ps.hk);
      ps.n = __builtin_amdgcn_readfirstlane(ps.n);
      return ps;
    }
  };

  // ---- per-lane constants ----
  const int lrow = lane >> 4, lslot = lane & 15;
  const int k_chunk = lslot ^ ((wave * 4 + lrow) & 15);
  const int v_chunk = lslot ^ (4 * lrow);
  const unsigned k_rb = lay.k_r * 2, v_rb = lay.v_r * 2;  // row strides in bytes
  const unsigned k_voff = (wave * 4 + lrow) * k_rb + k_chunk * 16;
  const unsigned v_voff = (wave * 4 + lrow) * v_rb + v_chunk * 16;
  typedef const __attribute__((address_space(3))) half8* lds_half8_t;
  unsigned k_frag[8], v_frag[4];  // LDS addresses of the fragment reads, opaque (see fa_fwd_d128_pipe)
  {
    const int kb0 = r32 * 256 + ((h ^ (lane & 15)) * 16);
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      k_frag[ks] = (unsigned)(uintptr_t)MI355_LDS(char, lds + (kb0 ^ (ks * 32)));
      asm volatile("" : "+v"(k_frag[ks]));
    }
    const int i16 = lane & 15, g16 = lane >> 4;
    const int v_row = 4 * (g16 >> 1) + (i16 >> 2);
    const int vb0 = VBUF + v_row * 256 + (i16 >> 2) * 64 + (2 * (g16 & 1) + ((i16 & 3) >> 1)) * 16 + (i16 & 1) * 8;
#pragma unroll
    for (int dt = 0; dt < 4; dt++) {
      v_frag[dt] = (unsigned)(uintptr_t)MI355_LDS(char, lds + (vb0 ^ (dt * 64)));
      asm volatile("" : "+v"(v_frag[dt]));
    }
  }

  half8 qf[8];
  // Q rows of pass ps: requested as they lie in memory (rows at or beyond Sq: zeros), later scaled by scale . log2(e),
  // rounded to the 16-bit format again and kept as the B operands of the score MFMAs
  auto request_q = [&](const Pass& ps, half8* raw) {
    const int ql = opaque_lane_id();  // (addresses derived from `lane` would be held in registers through the key walk)
    const int q_row = ps.qb * BLOCK_M + wave * 32 + (ql & 31);
    const half_t* qp = Q + ps.b * lay.q_b + ps.hq * lay.q_h + (size_t)q_row * lay.q_r + (ql >> 5) * 8;
    if (q_row < Sq) {
#pragma unroll
      for (int ks = 0; ks < 8; ks++) raw[ks] = *reinterpret_cast<const half8*>(qp + ks * 16);
    } else {
#pragma unroll
      for (int ks = 0; ks < 8; ks++)
#pragma unroll
        for (int e = 0; e < 8; e++) raw[ks][e] = (half_t)0;
    }
  };
  auto convert_q = [&](const half8* raw) {
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) qf[ks][e] = cvt16<BF>(to_f32<BF>(raw[ks][e]) * scale_log2e);
  };

  Pass cur = pass_at(0);
  if (cur.ord < 0) return;  // (the launcher starts no more workgroups than units)
  bool tiles_requested = false;  // K 0, K 1, V 0 of `cur` already requested (by the pass before)

  for (;;) {  // passes
  Pass nxt;  // looked up behind trip 0 (its divisions then run beside the other waves' work, not between two passes)
  nxt.ord = -1, nxt.b = nxt.hq = nxt.hk = nxt.qb = 0, nxt.n = 2;
  const int q0 = cur.qb * BLOCK_M;
  const int wq0 = q0 + wave * 32;
  const int q_row = wq0 + r32;
  const int n_tiles = cur.n;
  const half_t* Kb = K + cur.b * lay.k_b + cur.hk * lay.k_h;
  const half_t* Vb = V + cur.b * lay.v_b + cur.hk * lay.v_h;

  auto issue_kv = [&](const half_t* base, unsigned rb, unsigned voff, int tile, int lds_off) {
    char* dst = lds + lds_off + wave * 1024;
    const int row0 = tile * FA_BLOCK_N;
    int rem = Sk - row0;
    rem = rem > FA_BLOCK_N ? FA_BLOCK_N : rem;
    const buffer_rsrc_t rs = make_buffer(reinterpret_cast<const char*>(base) + (size_t)row0 * rb, (unsigned)(rem - 1) * rb + 256u);
#pragma unroll
    for (int i = 0; i < NI; i++) buffer_load_lds_16B(rs, voff + (unsigned)(i * NW * 4) * rb, 0, dst + i * NW * 1024);
  };

  floatx16 oacc[4];
#pragma unroll
  for (int dt = 0; dt < 4; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) oacc[dt][r] = 0.f;
  floatx16 negm;
#pragma unroll
  for (int r = 0; r < 16; r++) negm[r] = 0.f;
  float l_run = 0.f;
  float grow_thr = -INFINITY;
  constexpr float kRescaleThreshold = 8.f;

  auto wave_active = [&](int tile) { return !CAUSAL || (tile * FA_BLOCK_N <= wq0 + 31 + causal_off); };

  auto scores = [&](int koff, floatx16* s) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (int ks = 0; ks < 8; ks++) {
        half8 kf = *(lds_half8_t)(uintptr_t)(k_frag[ks] + (unsigned)(koff + t * 8192));
        s[t] = mfma16<BF>(kf, qf[ks], ks == 0 ? negm : s[t]);
      }
    }
  };

  // softmax of tile `tile` (scores in s) and O^T += V(slot)^T . P^T, with the scores of the following tile computed between
  // the exponentials; LAST: there is no following tile
  auto softmax_pv = [&](int tile, auto voff_tag, auto last_tag, floatx16* s, int koff_next, floatx16* s_next) {
    constexpr int VOFF = decltype(voff_tag)::value;
    constexpr bool LAST = decltype(last_tag)::value;
    {
      const int key0 = tile * FA_BLOCK_N;
      const bool need_mask = (CAUSAL && (key0 + FA_BLOCK_N - 1 > wq0 + causal_off)) || (key0 + FA_BLOCK_N > Sk);
      if (need_mask) {
        const int lim = CAUSAL ? (q_row + causal_off < Sk - 1 ? q_row + causal_off : Sk - 1) : Sk - 1;
        const int rel = lim - key0 - 4 * h;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const unsigned hide = (unsigned)((rel - (32 * t + 8 * (r >> 2) + (r & 3))) >> 31);
            const float sv = s[t][r];
            s[t][r] = __builtin_bit_cast(float, (hide & 0xFF800000u) | (~hide & __builtin_bit_cast(unsigned, sv)));
          }
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[t][r]);
    if (__builtin_amdgcn_ballot_w64(mx > grow_thr) != 0) {
      const float mxx = fmaxf(mx, __shfl_xor(mx, 32));
      const bool first = grow_thr == -INFINITY;
      const float delta = first ? (mxx == -INFINITY ? 0.f : mxx) : fmaxf(mxx, 0.f);
      const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(-delta);
      if (mxx != -INFINITY) grow_thr = kRescaleThreshold;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) oacc[dt][r] *= alpha;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) s[t][r] -= delta;
#pragma unroll
      for (int r = 0; r < 16; r++) negm[r] -= delta;
    }
    half8 pf[4];
    float psum = 0.f;
    // Scores of the next tile and the softmax of this one, step by step: score MFMA i, the K fragment of MFMA i + 3
    // requested, and the work of score pair i (two exponentials, one packed conversion, one dot2) behind it.  A
    // scheduling barrier after every step pins the order (a wave issues in order: only vector work placed between two
    // MFMAs runs while the first occupies the matrix pipe).
    __builtin_amdgcn_sched_barrier(0);
    {
      half8 kf[4];
      half2v pp_prev = {(half_t)0, (half_t)0};
      auto kread = [&](int i) { return *(lds_half8_t)(uintptr_t)(k_frag[i & 7] + (unsigned)(koff_next + (i >> 3) * 8192)); };
      if constexpr (!LAST) {
        kf[0] = kread(0);
        kf[1] = kread(1);
        kf[2] = kread(2);
      }
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int t = i >> 3, ks = i & 7, r = 2 * ks;
        if constexpr (!LAST) {
          if (i + 3 < 16) kf[(i + 3) & 3] = kread(i + 3);
          s_next[t] = mfma16<BF>(kf[i & 3], qf[ks], ks == 0 ? negm : s_next[t]);
        }
        // (the empty statement ties the pair's arithmetic to this step: without side effects of its own it is placed
        // wherever instruction selection likes, scheduling barriers or not)
        float e0 = __builtin_amdgcn_exp2f(s[t][r]), e1 = __builtin_amdgcn_exp2f(s[t][r + 1]);
        if (i > 0) psum = dot2_ones<BF>(pp_prev, psum);  // (one step behind its conversion, as in fa_fwd_d128_pipe)
        half2v pp = cvt16x2<BF>(e0, e1);
        asm volatile("" : "+v"(pp), "+v"(psum));
        pf[t * 2 + (r >> 3)][r & 7] = pp[0];
        pf[t * 2 + (r >> 3)][(r & 7) + 1] = pp[1];
        pp_prev = pp;
        __builtin_amdgcn_sched_barrier(0);
      }
      psum = dot2_ones<BF>(pp_prev, psum);
    }
    l_run += psum;
    half4 vlo[3], vhi[3];  // V^T reads and their waits in assembly, as in fa_fwd_d128_pipe
    auto vr = [&](auto itag) {
      constexpr int i = decltype(itag)::value;
      constexpr int off = VOFF + (i >> 2) * 4096;
      half4 &lo = vlo[i % 3], &hi = vhi[i % 3];
      const unsigned addr = v_frag[i & 3];
      asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                   : "=&v"(lo), "=&v"(hi)
                   : "v"(addr), "n"(off), "n"(off + 2048));
    };
    vr(std::integral_constant<int, 0>{});
    vr(std::integral_constant<int, 1>{});
    static_for<0, 16>([&](auto itag) {
      constexpr int i = decltype(itag)::value;
      if constexpr (i + 2 < 16) vr(std::integral_constant<int, i + 2>{});
      half4 &lo = vlo[i % 3], &hi = vhi[i % 3];
      if constexpr (i + 2 < 16)
        asm volatile("s_waitcnt lgkmcnt(4)" : "+v"(lo), "+v"(hi));
      else if constexpr (i + 1 < 16)
        asm volatile("s_waitcnt lgkmcnt(2)" : "+v"(lo), "+v"(hi));
      else
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(lo), "+v"(hi));
      const half8 vf = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      oacc[i & 3] = mfma16<BF>(vf, pf[i >> 2], oacc[i & 3]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  floatx16 sa[2], sb[2];
  if (!tiles_requested) {
    half8 raw[8];
    request_q(cur, raw);
    issue_kv(Kb, k_rb, k_voff, 0, 0);
    issue_kv(Vb, v_rb, v_voff, 0, VBUF);
    issue_kv(Kb, k_rb, k_voff, 1, TILE_B);
    convert_q(raw);
    wait_vmcnt0();
    __syncthreads();
  }
  scores(0, sa);  // every wave sees keys in a pass's first tile
  // trip 0 overwrites the K(0) slot with K(2): every wave must have read its K(0) fragments first
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __syncthreads();

  // trip j (PAR = j & 1): loads for K(j+2) and V(j+1); scores of tile j+1; softmax + PV of tile j
  auto trip = [&](auto par_tag, int j, floatx16* s_cur, floatx16* s_next) {
    constexpr int PAR = decltype(par_tag)::value;
    constexpr int K_CUR = PAR * TILE_B, K_NEXT = (1 - PAR) * TILE_B, V_CUR = PAR * TILE_B, V_NEXT = VBUF + (1 - PAR) * TILE_B;
    if (j + 2 < n_tiles) issue_kv(Kb, k_rb, k_voff, j + 2, K_CUR);
    if (j + 1 < n_tiles) issue_kv(Vb, v_rb, v_voff, j + 1, V_NEXT);
    if (wave_active(j)) softmax_pv(j, std::integral_constant<int, V_CUR>{}, std::false_type{}, s_cur, K_NEXT, s_next);  // idle from here on otherwise
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
  };
  // A pass of an even tile count runs its last tile (an odd trip) apart, behind the requests for the next pass: there are
  // no loads and no scores left for this pass, neither K slot is read again and V slot 0 was last read by the trip before.
  // A pass of an odd count ends with an ordinary trip and the requests follow it.
  const int n_plain = (n_tiles & 1) ? n_tiles : n_tiles - 1;
  for (int j = 0; j < n_plain; j += 2) {
    trip(std::integral_constant<int, 0>{}, j, sa, sb);
    if (j == 0) nxt = pass_at(cur.ord + 1);  // (two tiles at least: trip 0 is never the last)
    if (j + 1 < n_plain) trip(std::integral_constant<int, 1>{}, j + 1, sb, sa);
  }

  // ---- between passes ----
  half8 qraw[8];
  request_q(nxt.ord >= 0 ? nxt : cur, qraw);  // (unconditional, and converted unconditionally below: the old Q fragments are dead from here on)
  if (nxt.ord >= 0) {
    const half_t* Kn = K + nxt.b * lay.k_b + nxt.hk * lay.k_h;
    const half_t* Vn = V + nxt.b * lay.v_b + nxt.hk * lay.v_h;
    issue_kv(Kn, k_rb, k_voff, 0, 0);
    issue_kv(Vn, v_rb, v_voff, 0, VBUF);
    issue_kv(Kn, k_rb, k_voff, 1, TILE_B);
  }
  if (n_plain < n_tiles) {
    if (wave_active(n_tiles - 1)) softmax_pv(n_tiles - 1, std::integral_constant<int, TILE_B>{}, std::true_type{}, sb, 0, sa);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  const float l_tot = l_run + __shfl_xor(l_run, 32);
  const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;
  half8 orow[32 / 4];  // the rows this lane stores: 16-byte chunk ec of rows er, er + 4, ...
  const int el = opaque_lane_id();
  const int er = el >> 4, ec = el & 15;
  {
    // Output through the wave's staging region, STG_ROWS rows per round (chunk c of row r in slot c ^ (r & 15)): a lane
    // holds 4-value pieces of one row; whole 16-byte chunks are read back, to be stored as full rows
    char* ep = lds + STG + wave * (STG_ROWS * 256);
    const int e32 = el & 31, eh = el >> 5;
#pragma unroll
    for (int round = 0; round < 32 / STG_ROWS; round++) {
      if (STG_ROWS == 32 || (e32 / STG_ROWS) == round) {
#pragma unroll
        for (int dt = 0; dt < 4; dt++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const half4 v = {cvt16<BF>(oacc[dt][4 * q] * inv), cvt16<BF>(oacc[dt][4 * q + 1] * inv), cvt16<BF>(oacc[dt][4 * q + 2] * inv),
                             cvt16<BF>(oacc[dt][4 * q + 3] * inv)};
            *reinterpret_cast<half4*>(ep + (e32 % STG_ROWS) * 256 + (((dt * 4 + q) ^ (e32 & 15)) * 16) + 8 * eh) = v;
          }
      }
#pragma unroll
      for (int it = 0; it < STG_ROWS / 4; it++) {
        const int lr = it * 4 + er, row = round * STG_ROWS + lr;
        orow[round * (STG_ROWS / 4) + it] = *reinterpret_cast<const half8*>(ep + lr * 256 + ((ec ^ (row & 15)) * 16));
      }
    }
  }
  convert_q(qraw);  // (the oldest of the requests)
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the next pass's first tiles
  __syncthreads();
  {
    // the stores are left in flight: they drain under the next pass's first trip, whose closing wait covers them
    half_t* Ob = O + cur.b * lay.o_b + cur.hq * lay.o_h;
#pragma unroll
    for (int it = 0; it < 8; it++) {
      const int row = it * 4 + er;
      if (wq0 + row < Sq) *reinterpret_cast<half8*>(Ob + (size_t)(wq0 + row) * lay.o_r + ec * 8) = orow[it];
    }
  }
  if (nxt.ord < 0) break;
  tiles_requested = true;
  cur = nxt;
  }  // passes
}

static const char* kFaVariants[] = {"d128_bm128_bn64_w4_pipelined", "d128_bm128_bn64_w4", "d128_bm256_bn64_w8_pipelined",
                                    "d128_bm256_bn64_w8_walk", "d128_bm128_bn64_w4_walk", "d128_bm128_bn64_w4_m16",
                                    "d128_bm256_bn64_w8_m16"};
int fa_variant_count() { return 7; }
const char* fa_variant_name(int i) { return (i >= 0 && i < 7) ? kFaVariants[i] : nullptr; }

}  // namespace mi355

using namespace mi355;

// number of CUs of the current device (cached per device)
static int fa_cu_count() {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cached[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <bool BF>
static int fa_launch(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H, int64_t Hkv, int64_t Sq,
                     int64_t Sk, int64_t D, const FaLayout& lay, float scale, int is_causal, int variant, void* stream,
                     const char* who) {
  if (!q || !k || !v || !o) return fail(-MI355_E_NULL, "%s: null pointer", who);
  if (D != 128) return fail(-MI355_E_SHAPE, "%s: head dim %lld not supported (only 128)", who, (long long)D);
  if (B <= 0 || H <= 0 || Sq <= 0 || Sk <= 0 || B * H > (1 << 24) || Sq > (1 << 24) || Sk > (1 << 24))
    return fail(-MI355_E_SHAPE, "%s: bad shape B=%lld H=%lld Sq=%lld Sk=%lld", who, (long long)B, (long long)H, (long long)Sq,
                (long long)Sk);
  if (Hkv <= 0 || H % Hkv != 0)
    return fail(-MI355_E_SHAPE, "%s: %lld query heads over %lld key/value heads", who, (long long)H, (long long)Hkv);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return fail(-MI355_E_ALIGN, "%s: q, k, v, o must be 16-byte aligned", who);
  if (variant > 6) return fail(-MI355_E_DTYPE, "%s: variant %d out of range", who, variant);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be positive and finite", who);
  const int BH = (int)(B * H);
  const int q_blocks = (int)((Sq + FA_BLOCK_M - 1) / FA_BLOCK_M);
  const int lds_bytes = 2 * FA_STAGE;
  static std::atomic<uint64_t> lds_ok[4] = {};
  const void* kernels[4] = {reinterpret_cast<const void*>(fa_fwd_d128<true, BF>), reinterpret_cast<const void*>(fa_fwd_d128<false, BF>),
                            reinterpret_cast<const void*>(fa_fwd_d128_pipe<true, BF>),
                            reinterpret_cast<const void*>(fa_fwd_d128_pipe<false, BF>)};
  for (int i = 0; i < 4; i++)
    if (int rc = allow_lds(kernels[i], lds_bytes, lds_ok[i], "fa_fwd_d128")) return rc;
  const float scale_log2e = scale * 1.4426950408889634f;
  // Without a mask, and with enough 256-query blocks for every CU, the 8-wave form is ahead (2 x 32 x 4096: 503 against
  // 514 us); with the causal mask the two are level and the 4-wave form has the finer-grained tail.
  // The automatic choice is the 16x16x32 form: eight waves (with the exponentials spread into the output MFMAs) for
  // unmasked shapes with enough 256-query blocks for every CU (2 x 32 x 4096: 475 us against 483 for the 32x32x16 form
  // on the same box), four waves otherwise (causal 2 x 32 x 4096: 263 against 269; the finer-grained tail).
  if (variant < 0) variant = (!is_causal && (int64_t)BH * ((Sq + 255) / 256) >= 512) ? 6 : 5;
  if (variant == 5 || variant == 6) {
    // the pipelined forms on 16x16x32 MFMAs, 4 waves (128-query blocks) or 8 (256)
    const bool w8 = variant == 6;
    const int bm = w8 ? 256 : 128;
    const int qbm = (int)((Sq + bm - 1) / bm);
    const void* kern = w8 ? (is_causal ? (const void*)fa_fwd_d128_m16<true, BF, 8, true> : (const void*)fa_fwd_d128_m16<false, BF, 8, true>)
                          : (is_causal ? (const void*)fa_fwd_d128_m16<true, BF, 4, false> : (const void*)fa_fwd_d128_m16<false, BF, 4, false>);
    static std::atomic<uint64_t> okm[4] = {};
    if (int rc = allow_lds(kern, lds_bytes, okm[(w8 ? 2 : 0) + (is_causal ? 1 : 0)], "fa_fwd_d128_m16")) return rc;
    dim3 grid(BH * (is_causal ? (qbm + 1) / 2 : qbm)), block(w8 ? 512 : 256);
    const half_t *qp = (const half_t*)q, *kp = (const half_t*)k, *vp = (const half_t*)v;
    half_t* op = (half_t*)o;
    int bh_i = BH, sq_i = (int)Sq, sk_i = (int)Sk, qb_i = qbm;
    FaLayout lay_v = lay;
    float sc = scale_log2e;
    FaPaged no_pages{nullptr, nullptr, 0, 0, 0};
    void* args[] = {&qp, &kp, &vp, &op, &bh_i, &sq_i, &sk_i, &sc, &qb_i, &lay_v, &no_pages};
    hipError_t e = hipLaunchKernel(kern, grid, block, args, lds_bytes, reinterpret_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail((int)e, "%s: launch of fa_fwd_d128_m16 failed: %s", who, hipGetErrorString(e));
    return check_launch("fa_fwd_d128_m16", grid, block, lds_bytes);
  }
  if (variant == 3 || variant == 4) {
    // the persistent forms: every pass needs two key tiles, and the masked form a square mask (no pass without keys)
    const bool w8 = variant == 3;
    const int bm = w8 ? 256 : 128;
    const int qbw = (int)((Sq + bm - 1) / bm);
    const int64_t units_w = (int64_t)BH * (is_causal ? (qbw + 1) / 2 : qbw);
    if (Sk < 128 || (is_causal && Sq != Sk) || units_w >= (1ll << 30))
      return fail(-MI355_E_SHAPE, "%s: the persistent form needs Sk >= 128%s (Sq=%lld Sk=%lld)", who, is_causal ? " and Sq == Sk" : "",
                  (long long)Sq, (long long)Sk);
    const void* kern = w8 ? (is_causal ? (const void*)fa_fwd_d128_walk<true, BF, 8> : (const void*)fa_fwd_d128_walk<false, BF, 8>)
                          : (is_causal ? (const void*)fa_fwd_d128_walk<true, BF, 4> : (const void*)fa_fwd_d128_walk<false, BF, 4>);
    static std::atomic<uint64_t> okw[4] = {};
    const int ldsw = 4 * FA_BLOCK_N * 256 + (w8 ? 8 * 8192 : 4 * 2048);  // K and V rings + output staging
    if (int rc = allow_lds(kern, ldsw, okw[(w8 ? 2 : 0) + (is_causal ? 1 : 0)], "fa_fwd_d128_walk")) return rc;
    int g = fa_cu_count() * (w8 ? 1 : 2);  // workgroups resident at once
    if (((BH / lay.group) & 7) == 0) g &= ~7;  // units of one K/V head stay on the XCD that a workgroup runs on
    if (g < 1) g = 1;
    if (units_w < g) g = (int)units_w;
    dim3 grid(g), block(w8 ? 512 : 256);
    const half_t *qp = (const half_t*)q, *kp = (const half_t*)k, *vp = (const half_t*)v;
    half_t* op = (half_t*)o;
    int bh_i = BH, sq_i = (int)Sq, sk_i = (int)Sk;
    FaLayout lay_v = lay;
    float sc = scale_log2e;
    int qb_i = qbw;
    void* args[] = {&qp, &kp, &vp, &op, &bh_i, &sq_i, &sk_i, &sc, &qb_i, &lay_v};
    hipError_t e = hipLaunchKernel(kern, grid, block, args, ldsw, reinterpret_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail((int)e, "%s: launch of fa_fwd_d128_walk failed: %s", who, hipGetErrorString(e));
    return check_launch("fa_fwd_d128_walk", grid, block, ldsw);
  }
  if (variant == 2) {
    // eight waves: 256-query blocks, one workgroup per CU
    auto kern = is_causal ? fa_fwd_d128_pipe<true, BF, 8> : fa_fwd_d128_pipe<false, BF, 8>;
    static std::atomic<uint64_t> ok8[2] = {};
    const int lds8 = lds_bytes;
    if (int rc = allow_lds(reinterpret_cast<const void*>(kern), lds8, ok8[is_causal ? 1 : 0], "fa_fwd_d128_pipe<8>")) return rc;
    const int qb8 = (int)((Sq + 255) / 256);
    dim3 grid(BH * (is_causal ? (qb8 + 1) / 2 : qb8)), block(512);
    hipLaunchKernelGGL(kern, grid, block, lds8, reinterpret_cast<hipStream_t>(stream), (const half_t*)q, (const half_t*)k,
                       (const half_t*)v, (half_t*)o, BH, (int)Sq, (int)Sk, scale_log2e, qb8, lay);
    return check_launch("fa_fwd_d128_pipe<8 waves>", grid, block, lds8);
  }
  // the pipelined causal kernel takes a pair of query blocks per workgroup
  const int units = (variant != 1 && is_causal) ? (q_blocks + 1) / 2 : q_blocks;
  dim3 grid(BH * units), block(256);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (variant == 1) {
    auto kern = is_causal ? fa_fwd_d128<true, BF> : fa_fwd_d128<false, BF>;
    hipLaunchKernelGGL(kern, grid, block, lds_bytes, s, (const half_t*)q, (const half_t*)k, (const half_t*)v, (half_t*)o, BH,
                       (int)Sq, (int)Sk, scale_log2e, q_blocks, lay);
  } else {
    auto kern = is_causal ? fa_fwd_d128_pipe<true, BF> : fa_fwd_d128_pipe<false, BF>;
    hipLaunchKernelGGL(kern, grid, block, lds_bytes, s, (const half_t*)q, (const half_t*)k, (const half_t*)v, (half_t*)o, BH,
                       (int)Sq, (int)Sk, scale_log2e, q_blocks, lay);
  }
  return check_launch(variant == 1 ? "fa_fwd_d128" : "fa_fwd_d128_pipe", grid, block, lds_bytes);
}

template <bool BF>
static int fa_contiguous(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H, int64_t Sq, int64_t Sk,
                         int64_t D, float scale, int is_causal, int variant, void* stream) {
  FaLayout lay;
  lay.q_b = H * Sq * 128, lay.q_h = Sq * 128, lay.q_r = 128;
  lay.o_b = lay.q_b, lay.o_h = lay.q_h, lay.o_r = 128;
  lay.k_b = lay.v_b = H * Sk * 128, lay.k_h = lay.v_h = Sk * 128, lay.k_r = lay.v_r = 128;
  lay.H = (int)H, lay.group = 1;
  return fa_launch<BF>(q, k, v, o, B, H, H, Sq, Sk, D, lay, scale, is_causal, variant, stream,
                       BF ? "flash_attn_fwd_bf16" : "flash_attn_fwd");
}

extern "C" int mi355_flash_attn_fwd(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H, int64_t Sq,
                                    int64_t Sk, int64_t D, float scale, int is_causal, int variant, void* stream) {
  return fa_contiguous<false>(q, k, v, o, B, H, Sq, Sk, D, scale, is_causal, variant, stream);
}

extern "C" int mi355_flash_attn_fwd_bf16(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H, int64_t Sq,
                                         int64_t Sk, int64_t D, float scale, int is_causal, int variant, void* stream) {
  return fa_contiguous<true>(q, k, v, o, B, H, Sq, Sk, D, scale, is_causal, variant, stream);
}

template <bool BF>
static int fa_strided(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H, int64_t Hkv, int64_t Sq,
                      int64_t Sk, int64_t D, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                      const int64_t* o_strides, float scale, int is_causal, int variant, void* stream) {
  const char* who = BF ? "flash_attn_fwd_strided_bf16" : "flash_attn_fwd_strided";
  if (!q_strides || !k_strides || !v_strides || !o_strides) return fail(-MI355_E_NULL, "%s: null stride array", who);
  const int64_t* all[4] = {q_strides, k_strides, v_strides, o_strides};
  for (const int64_t* st : all) {
    for (int i = 0; i < 3; i++)
      if (st[i] < 0 || (st[i] & 7)) return fail(-MI355_E_ALIGN, "%s: strides must be non-negative multiples of 8 elements", who);
    if (st[2] < 128 || st[2] >= (1ll << 24))
      return fail(-MI355_E_SHAPE, "%s: row stride %lld outside [128, 2^24)", who, (long long)st[2]);
  }
  if ((B > 1 && o_strides[0] == 0) || (H > 1 && o_strides[1] == 0)) return fail(-MI355_E_SHAPE, "%s: output batch / head strides must not be 0", who);
  FaLayout lay;
  lay.q_b = q_strides[0], lay.q_h = q_strides[1], lay.q_r = (unsigned)q_strides[2];
  lay.k_b = k_strides[0], lay.k_h = k_strides[1], lay.k_r = (unsigned)k_strides[2];
  lay.v_b = v_strides[0], lay.v_h = v_strides[1], lay.v_r = (unsigned)v_strides[2];
  lay.o_b = o_strides[0], lay.o_h = o_strides[1], lay.o_r = (unsigned)o_strides[2];
  lay.H = (int)H, lay.group = Hkv > 0 ? (int)(H / Hkv) : 1;
  return fa_launch<BF>(q, k, v, o, B, H, Hkv, Sq, Sk, D, lay, scale, is_causal, variant, stream, who);
}

extern "C" int mi355_flash_attn_fwd_strided(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H,
                                            int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, const int64_t* q_strides,
                                            const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                            float scale, int is_causal, int variant, void* stream) {
  return fa_strided<false>(q, k, v, o, B, H, Hkv, Sq, Sk, D, q_strides, k_strides, v_strides, o_strides, scale, is_causal, variant,
                           stream);
}

extern "C" int mi355_flash_attn_fwd_strided_bf16(const void* q, const void* k, const void* v, void* o, int64_t B, int64_t H,
                                                 int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, const int64_t* q_strides,
                                                 const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                                                 float scale, int is_causal, int variant, void* stream) {
  return fa_strided<true>(q, k, v, o, B, H, Hkv, Sq, Sk, D, q_strides, k_strides, v_strides, o_strides, scale, is_causal, variant,
                          stream);
}

template <bool BF>
static int fa_paged_prefill(const void* q, const void* k_cache, const void* v_cache, const void* block_table, const void* seq_lens,
                            void* out, int64_t num_seqs, int64_t num_new, int64_t num_q_heads, int64_t num_kv_heads, int64_t D,
                            int64_t page_size, int64_t max_pages_per_seq, int64_t num_pages, float scale, void* stream) {
  const char* who = BF ? "paged_prefill_attn_bf16" : "paged_prefill_attn";
  if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out) return fail(-MI355_E_NULL, "%s: null pointer", who);
  if (D != 128) return fail(-MI355_E_SHAPE, "%s: head dim %lld not supported (only 128)", who, (long long)D);
  int page_shift = -1;
  for (int sh = 0; sh <= 4; sh++)
    if (page_size == (16ll << sh)) page_shift = sh;
  if (page_shift < 0) return fail(-MI355_E_SHAPE, "%s: page size %lld not supported (16, 32, 64, 128 or 256)", who, (long long)page_size);
  if (num_seqs <= 0 || num_new <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_pages_per_seq <= 0 || num_pages <= 0 ||
      num_seqs * num_q_heads > (1 << 24) || num_new > (1 << 20) || max_pages_per_seq > (1 << 20) || num_pages > (1 << 24) ||
      (max_pages_per_seq * page_size) > (1 << 24))
    return fail(-MI355_E_SHAPE, "%s: bad shape seqs=%lld new=%lld q_heads=%lld kv_heads=%lld max_pages=%lld pages=%lld", who,
                (long long)num_seqs, (long long)num_new, (long long)num_q_heads, (long long)num_kv_heads,
                (long long)max_pages_per_seq, (long long)num_pages);
  if (num_q_heads % num_kv_heads != 0)
    return fail(-MI355_E_SHAPE, "%s: %lld query heads over %lld key/value heads", who, (long long)num_q_heads, (long long)num_kv_heads);
  if (num_kv_heads * 128 >= (1 << 24)) return fail(-MI355_E_SHAPE, "%s: too many key/value heads", who);
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out))
    return fail(-MI355_E_ALIGN, "%s: q, k_cache, v_cache, out must be 16-byte aligned", who);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be positive and finite", who);
  FaLayout lay;
  lay.q_b = num_new * num_q_heads * 128, lay.q_h = 128, lay.q_r = (unsigned)(num_q_heads * 128);
  lay.o_b = lay.q_b, lay.o_h = 128, lay.o_r = lay.q_r;
  lay.k_b = lay.v_b = 0, lay.k_h = lay.v_h = 128, lay.k_r = lay.v_r = (unsigned)(num_kv_heads * 128);
  lay.H = (int)num_q_heads, lay.group = (int)(num_q_heads / num_kv_heads);
  const int BH = (int)(num_seqs * num_q_heads);
  const int q_blocks = (int)((num_new + FA_BLOCK_M - 1) / FA_BLOCK_M);
  const int lds_bytes = 2 * FA_STAGE;
  auto kern = fa_fwd_d128_m16<true, BF, 4, false, FaForm::PAGED>;
  static std::atomic<uint64_t> lds_ok{0};
  if (int rc = allow_lds(reinterpret_cast<const void*>(kern), lds_bytes, lds_ok, "fa_fwd_d128_m16<paged>")) return rc;
  dim3 grid(BH * ((q_blocks + 1) / 2)), block(256);
  const FaPaged pg{static_cast<const int*>(block_table), static_cast<const int*>(seq_lens), (int)max_pages_per_seq, (int)num_pages,
                   page_shift};
  hipLaunchKernelGGL(kern, grid, block, lds_bytes, reinterpret_cast<hipStream_t>(stream), (const half_t*)q, (const half_t*)k_cache,
                     (const half_t*)v_cache, (half_t*)out, BH, (int)num_new, 0, scale * 1.4426950408889634f, q_blocks, lay, pg);
  return check_launch("fa_fwd_d128_m16<paged>", grid, block, lds_bytes);
}

extern "C" int mi355_paged_prefill_attn(const void* q, const void* k_cache, const void* v_cache, const void* block_table,
                                        const void* seq_lens, void* out, int64_t num_seqs, int64_t num_new, int64_t num_q_heads,
                                        int64_t num_kv_heads, int64_t D, int64_t page_size, int64_t max_pages_per_seq,
                                        int64_t num_pages, float scale, void* stream) {
  return fa_paged_prefill<false>(q, k_cache, v_cache, block_table, seq_lens, out, num_seqs, num_new, num_q_heads, num_kv_heads, D,
                                 page_size, max_pages_per_seq, num_pages, scale, stream);
}

extern "C" int mi355_paged_prefill_attn_bf16(const void* q, const void* k_cache, const void* v_cache, const void* block_table,
                                             const void* seq_lens, void* out, int64_t num_seqs, int64_t num_new,
                                             int64_t num_q_heads, int64_t num_kv_heads, int64_t D, int64_t page_size,
                                             int64_t max_pages_per_seq, int64_t num_pages, float scale, void* stream) {
  return fa_paged_prefill<true>(q, k_cache, v_cache, block_table, seq_lens, out, num_seqs, num_new, num_q_heads, num_kv_heads, D,
                                page_size, max_pages_per_seq, num_pages, scale, stream);
}

namespace mi355 {

// The tree form's launch: arguments checked by the caller (paged_tree.hip).
template <bool BF, int QG>
static int fa_tree_launch(const TreeArgs& a, int num_seqs, hipStream_t stream) {
  auto kern = fa_fwd_d128_m16<false, BF, 4, false, FaForm::TREE, QG>;
  constexpr int block_m = 64 * QG;
  const int lds_bytes = 2 * FA_STAGE + block_m * (int)sizeof(unsigned long long) + 16;
  static std::atomic<uint64_t> lds_ok{0};
  if (int rc = allow_lds(reinterpret_cast<const void*>(kern), lds_bytes, lds_ok, "fa_fwd_d128_m16<tree>")) return rc;
  const int hq = a.num_kv_heads * a.group;
  FaLayout lay{};
  lay.q_b = lay.o_b = (int64_t)a.nodes * hq * 128, lay.q_h = lay.o_h = 128, lay.q_r = lay.o_r = (unsigned)(hq * 128);
  lay.k_h = lay.v_h = 128, lay.k_r = lay.v_r = (unsigned)(a.num_kv_heads * 128);
  lay.H = hq, lay.group = a.group;
  FaTree tr;
  tr.block_table = a.table, tr.seq_lens = a.seq_lens, tr.max_pages = a.max_pages, tr.num_pages = a.num_pages, tr.page_shift = a.page_shift;
  tr.parents = a.parents, tr.part_acc = a.part_acc, tr.part_ml = a.part_ml, tr.nodes = a.nodes, tr.num_kv_heads = a.num_kv_heads;
  tr.num_seqs = num_seqs, tr.num_splits = a.num_splits, tr.per_half = a.per_half;
  tr.row_blocks = (a.nodes * a.group + block_m - 1) / block_m;
  const int64_t wgs = (int64_t)num_seqs * a.num_splits * a.num_kv_heads * tr.row_blocks;
  if (wgs >= (1ll << 24)) return fail(-MI355_E_SHAPE, "paged_tree_attn: too many workgroups");  // 2^32 threads
  dim3 grid((unsigned)wgs), block(256);
  hipLaunchKernelGGL(kern, grid, block, lds_bytes, stream, a.q, a.kc, a.vc, a.out, 0, 0, 0, a.scale_log2e, 0, lay, tr);
  return check_launch("fa_fwd_d128_m16<tree>", grid, block, lds_bytes);
}
int fa_tree(const TreeArgs& a, int num_seqs, bool bf16, hipStream_t stream) {
  if (a.nodes * a.group <= 64) return bf16 ? fa_tree_launch<true, 1>(a, num_seqs, stream) : fa_tree_launch<false, 1>(a, num_seqs, stream);
  return bf16 ? fa_tree_launch<true, 2>(a, num_seqs, stream) : fa_tree_launch<false, 2>(a, num_seqs, stream);
}

}  // namespace mi355

// How a packed call is laid out.  The lengths are known on the device only; sizes are what decides.
struct FaVarlenPlan { int qg, pairs, ranked, chunks; };
static FaVarlenPlan fa_varlen_plan(int64_t num_seqs, int64_t total_q, int64_t total_k, int64_t H, int64_t Hkv, int is_causal) {
  FaVarlenPlan p;
  const int64_t rows = total_q * (H / Hkv), blocks = rows / FA_BLOCK_M * Hkv;
  // With the mask, a pair of blocks (the i-th from the end and the i-th from the start) is the same work everywhere in a sequence,
  // and half as many workgroups; where even single blocks would not fill the chip twice (512 workgroups are resident), they
  // are handed out singly.
  p.pairs = is_causal && blocks >= 2048;
  // Blocks of 64 rows where those of 128 would not fill the chip: twice the workgroups, each with half the work per key tile.
  // One prompt of 1024 tokens (32 query heads over 8) 23 against 29 us, 32 of 16 tokens 8.0 against 9.7; where the chip
  // is full the 64-row blocks are bound by LDS reads: 8 prompts of 256 tokens 22 against 20, one of 4096 164 against 134.
  p.qg = blocks < 512 ? 1 : 2;
  // Ranking costs every workgroup some 12 ns per sequence: worth it where sequences are long or few (32 of 2 to 600 tokens, 16
  // heads over one, 22.9 against 25.7 us, 16 of them 15.7 against 16.6; 64 of 2 to 100 tokens, 32 heads over 8, 21.3 against 18.0).
  p.ranked = num_seqs > 1 && num_seqs <= 64 && total_k / num_seqs >= 3 * num_seqs;
  // Few blocks that walk many keys: the number of chunks whose estimate is the smallest, in us: 3.5 for a workgroup and 0.85 for
  // each of its key tiles, twice and more where there are more workgroups than the 512 resident ones; and for the
  // joining 4 and the partial results written and read at 3.5 TB/s.  One to four sequences of 8192 keys and up to 128 new
  // tokens 116-134 us without, 20-92 with; 4 x 128 tokens in front of 1024 keys (16 query heads over 1) 20 without, 25 with 4.
  p.chunks = 1;
  if (p.qg == 1 && num_seqs <= 64) {
    const double full = (double)(rows / 64 + num_seqs) * Hkv / 512, tiles = (double)total_k / num_seqs / FA_BLOCK_N;
    double best = 0;
    for (int c = 1; c <= FA_MAX_CHUNKS; c++) {
      if (c > 1 && tiles < FA_MIN_CHUNK * c) break;
      const double t = (full * c > 1 ? full * c : 1.0) * (3.5 + 0.85 * tiles / c) + (c > 1 ? 4 + (double)total_q * H * c * 1040 / 3.5e6 : 0.0);
      if (c == 1 || t < best) best = t, p.chunks = c;
    }
  }
  return p;
}
static int64_t fa_varlen_scratch(const FaVarlenPlan& p, int64_t total_q, int64_t H) {
  return p.chunks == 1 ? 0 : total_q * H * p.chunks * (128 + 2) * (int64_t)sizeof(float);
}

template <bool BF>
static int fa_varlen(const void* q, const void* k, const void* v, void* o, const int32_t* cu_q, const int32_t* cu_k, int64_t num_seqs,
                     int64_t total_q, int64_t total_k, int64_t H, int64_t Hkv, int64_t D, const int64_t* q_strides,
                     const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides, float scale, int is_causal,
                     int zero_rest, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = BF ? "flash_attn_varlen_fwd_bf16" : "flash_attn_varlen_fwd";
  if (!q || !k || !v || !o || !cu_q || !cu_k || !q_strides || !k_strides || !v_strides || !o_strides)
    return fail(-MI355_E_NULL, "%s: null pointer", who);
  if (D != 128) return fail(-MI355_E_SHAPE, "%s: head dim %lld not supported (only 128)", who, (long long)D);
  if (num_seqs <= 0 || num_seqs > 65535 || total_q <= 0 || total_k <= 0 || total_q > (1 << 24) || total_k > (1 << 24) || H <= 0 ||
      H > 65535)
    return fail(-MI355_E_SHAPE, "%s: bad sizes seqs=%lld total_q=%lld total_k=%lld H=%lld", who, (long long)num_seqs,
                (long long)total_q, (long long)total_k, (long long)H);
  if (Hkv <= 0 || H % Hkv != 0)
    return fail(-MI355_E_SHAPE, "%s: %lld query heads over %lld key/value heads", who, (long long)H, (long long)Hkv);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return fail(-MI355_E_ALIGN, "%s: q, k, v, o must be 16-byte aligned", who);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be positive and finite", who);
  const int64_t* all[4] = {q_strides, k_strides, v_strides, o_strides};
  for (const int64_t* st : all) {  // {token, head}
    if (st[0] < 0 || st[1] < 0 || ((st[0] | st[1]) & 7))
      return fail(-MI355_E_ALIGN, "%s: strides must be non-negative multiples of 8 elements", who);
    if (st[0] < 128 || st[0] >= (1ll << 24) || st[1] >= (1ll << 40))
      return fail(-MI355_E_SHAPE, "%s: token stride %lld outside [128, 2^24)", who, (long long)st[0]);
  }
  if (H > 1 && o_strides[1] == 0) return fail(-MI355_E_SHAPE, "%s: the output's head stride must not be 0", who);
  FaLayout lay;
  lay.q_b = lay.k_b = lay.v_b = lay.o_b = 0;
  lay.q_h = q_strides[1], lay.q_r = (unsigned)q_strides[0];
  lay.k_h = k_strides[1], lay.k_r = (unsigned)k_strides[0];
  lay.v_h = v_strides[1], lay.v_r = (unsigned)v_strides[0];
  lay.o_h = o_strides[1], lay.o_r = (unsigned)o_strides[0];
  lay.H = (int)H, lay.group = (int)(H / Hkv);
  const int64_t group = H / Hkv, rows = total_q * group;
  if (rows > (1ll << 30)) return fail(-MI355_E_SHAPE, "%s: %lld query rows per key/value head, at most 2^30", who, (long long)rows);
  int group_shift = -1;
  for (int sh = 0; sh < 16; sh++)
    if (group == (1ll << sh)) group_shift = sh;
  FaVarlenPlan plan = fa_varlen_plan(num_seqs, total_q, total_k, H, Hkv, is_causal);
  if (!workspace || workspace_bytes < fa_varlen_scratch(plan, total_q, H)) plan.chunks = 1;
  if (plan.chunks > 1 && !aligned16(workspace)) return fail(-MI355_E_ALIGN, "%s: workspace must be 16-byte aligned", who);
  const int qg = plan.qg, block_m = 64 * qg;
  float* part = plan.chunks > 1 ? (float*)workspace : nullptr;
  const FaVarlen vl{cu_q, cu_k, (int)num_seqs, (int)total_q, (int)total_k, group_shift, zero_rest, plan.pairs, plan.ranked, plan.chunks, part,
                    part ? part + total_q * H * plan.chunks * 128 : nullptr};
  // the lengths are known on the device only: as many units as num_seqs sequences of total_q tokens can have
  const int64_t units = rows / (block_m << plan.pairs) + num_seqs;
  if (units * Hkv * plan.chunks >= (1ll << 24)) return fail(-MI355_E_SHAPE, "%s: too many query blocks", who);  // 2^32 threads
  const bool cut = plan.chunks > 1;
  auto kern = cut       ? (is_causal ? fa_fwd_d128_m16<true, BF, 4, false, FaForm::CHUNKED, 1> : fa_fwd_d128_m16<false, BF, 4, false, FaForm::CHUNKED, 1>)
              : qg == 1 ? (is_causal ? fa_fwd_d128_m16<true, BF, 4, false, FaForm::VARLEN, 1> : fa_fwd_d128_m16<false, BF, 4, false, FaForm::VARLEN, 1>)
                        : (is_causal ? fa_fwd_d128_m16<true, BF, 4, false, FaForm::VARLEN, 2> : fa_fwd_d128_m16<false, BF, 4, false, FaForm::VARLEN, 2>);
  const int lds_bytes = 2 * FA_STAGE + 16;
  static std::atomic<uint64_t> lds_ok[6] = {};
  if (int rc = allow_lds(reinterpret_cast<const void*>(kern), lds_bytes, lds_ok[(is_causal ? 1 : 0) + 2 * (cut ? 2 : qg - 1)], "fa_fwd_d128_m16<varlen>")) return rc;
  dim3 grid((unsigned)(units * Hkv * plan.chunks)), block(256);
  hipStream_t on = reinterpret_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(kern, grid, block, lds_bytes, on, (const half_t*)q, (const half_t*)k, (const half_t*)v, (half_t*)o, (int)H, 0, 0,
                     scale * 1.4426950408889634f, 0, lay, vl);
  int rc = check_launch("fa_fwd_d128_m16<varlen>", grid, block, lds_bytes);
  if (rc || !cut) return rc;
  dim3 join((unsigned)((total_q * H + 7) / 8));
  hipLaunchKernelGGL(fa_varlen_join<BF>, join, block, 0, on, vl, lay, (half_t*)o, is_causal);
  return check_launch("fa_varlen_join", join, block, 0);
}

extern "C" int64_t mi355_flash_attn_varlen_workspace_bytes(int64_t num_seqs, int64_t total_q, int64_t total_k, int64_t H, int64_t Hkv,
                                                          int is_causal) {
  if (num_seqs <= 0 || num_seqs > 65535 || total_q <= 0 || total_k <= 0 || total_q > (1 << 24) || total_k > (1 << 24) || H <= 0 ||
      H > 65535 || Hkv <= 0 || H % Hkv != 0)
    return 0;
  return fa_varlen_scratch(fa_varlen_plan(num_seqs, total_q, total_k, H, Hkv, is_causal), total_q, H);
}

extern "C" int mi355_flash_attn_varlen_fwd(const void* q, const void* k, const void* v, void* o, const int32_t* cu_seqlens_q,
                                           const int32_t* cu_seqlens_k, int64_t num_seqs, int64_t total_q, int64_t total_k, int64_t H,
                                           int64_t Hkv, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                           const int64_t* v_strides, const int64_t* o_strides, float scale, int is_causal,
                                           int zero_rest, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype == MI355_BF16)
    return fa_varlen<true>(q, k, v, o, cu_seqlens_q, cu_seqlens_k, num_seqs, total_q, total_k, H, Hkv, D, q_strides, k_strides, v_strides,
                           o_strides, scale, is_causal, zero_rest, workspace, workspace_bytes, stream);
  if (dtype == MI355_F16)
    return fa_varlen<false>(q, k, v, o, cu_seqlens_q, cu_seqlens_k, num_seqs, total_q, total_k, H, Hkv, D, q_strides, k_strides, v_strides,
                            o_strides, scale, is_causal, zero_rest, workspace, workspace_bytes, stream);
  return fail(-MI355_E_DTYPE, "flash_attn_varlen_fwd: dtype %d (MI355_F16 or MI355_BF16)", dtype);
}
