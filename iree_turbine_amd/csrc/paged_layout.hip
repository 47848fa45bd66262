// Block tables and slot maps of a batch step, built on the device from per-sequence lengths.
//
// Sequence s has c = context_lens[s] tokens in the cache and adds n = new_lens[s].  With p tokens per page its pages
// [ceil(c / p), ceil((c + n) / p)) are new and come from the front of the free list, in sequence order; every new token
// gets a row of the flat arrays: its sequence, position, and slot = table[s][pos / p] * p + pos % p.
//
// The work is a few bytes per token and sequence: the call is bound by launch and memory latency, so it is ONE launch
// without workspace.  Every workgroup owns PL_ROWS rows of the flat arrays and scans the lengths of the sequences
// itself (up to the one that fills its rows), instead of waiting for a scan kernel; workgroup 0 scans all of them and
// writes the per-sequence results (64 sequences of one new token 5.0 us, 1000 sequences and 26000 rows 6.8 us, of which an
// empty launch is 3.6).  No workgroup reads a table entry that another one writes: a new page's id follows
// from the scan, and the entry is written by the row of the page's first token.
#include "common.hpp"

namespace mi355 {

constexpr int PL_THREADS = 1024;
constexpr int PL_ROWS = 1024;  // rows of the flat arrays per workgroup, one per thread

// Inclusive prefix sum over the workgroup; `tmp` holds one value per wave; `total` is the sum of all.
__device__ __forceinline__ long long pl_scan(long long v, long long* tmp, long long& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  long long base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < PL_THREADS / 64; w++) {
    const long long t = tmp[w];
    base += w < wave ? t : 0;
    total += t;
  }
  __syncthreads();
  return v + base;
}

__global__ __launch_bounds__(PL_THREADS) void paged_layout_kernel(
    int* __restrict__ table, const int* __restrict__ context_lens, const int* __restrict__ new_lens,
    const int* __restrict__ free_pages, int num_free, int num_seqs, int max_pages, int page_bits, int num_rows,
    int* __restrict__ seq_lens, int* __restrict__ cu_new, int* __restrict__ positions, int* __restrict__ seq_ids,
    long long* __restrict__ slots, int* __restrict__ pages_needed) {
  __shared__ long long tmp[PL_THREADS / 64];
  // what a row has to know about its sequence, kept at the first of the workgroup's rows that belongs to it
  __shared__ int m_seq[PL_ROWS], m_skip[PL_ROWS], m_ctx[PL_ROWS], m_first[PL_ROWS];
  __shared__ int wave_top[PL_THREADS / 64];
  const int t = threadIdx.x;
  const int row0 = blockIdx.x * PL_ROWS;
  const int row1 = num_rows - row0 > PL_ROWS ? row0 + PL_ROWS : num_rows;
  const bool lead = blockIdx.x == 0;
  const int page = 1 << page_bits;
  m_seq[t] = -1;
  __syncthreads();

  long long rows_before = 0, pages_before = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += PL_THREADS) {
    const int s = s0 + t;
    long long c = 0, want = 0;
    if (s < num_seqs) {
      c = context_lens[s];
      want = new_lens[s];
      c = c < 0 ? 0 : c;
      want = want < 0 ? 0 : want;
    }
    long long all;
    const long long end = rows_before + pl_scan(want, tmp, all);
    const long long begin = end - want;
    // rows behind the last one there is are not admitted
    const long long b = begin < num_rows ? begin : num_rows, e = end < num_rows ? end : num_rows;
    const long long n = e - b;
    long long have = (c + page - 1) >> page_bits, upto = (c + n + page - 1) >> page_bits;
    have = have < max_pages ? have : max_pages;
    upto = upto < max_pages ? upto : max_pages;
    const long long fresh = s < num_seqs ? upto - have : 0;
    long long all_pages;
    const long long first = pages_before + pl_scan(fresh, tmp, all_pages) - fresh;
    if (s < num_seqs) {
      if (lead) {
        const long long len = c + n;
        seq_lens[s] = (int)(len < 0x7fffffffll ? len : 0x7fffffffll);
        cu_new[s + 1] = (int)e;
        if (s == 0) cu_new[0] = 0;
      }
      const long long lo = b > row0 ? b : row0, hi = e < row1 ? e : row1;
      if (lo < hi) {
        const int at = (int)(lo - row0);
        m_seq[at] = s;
        m_skip[at] = (int)(lo - b);  // tokens of the sequence in front of this workgroup's rows
        m_ctx[at] = (int)c;
        m_first[at] = (int)(first - have);  // free-list index of page 0, if all pages were new
      }
    }
    rows_before += all;
    pages_before += all_pages;
    if (!lead && rows_before >= row1) break;  // uniform: every thread has the same totals
  }
  if (lead && t == 0) *pages_needed = (int)(pages_before < 0x7fffffffll ? pages_before : 0x7fffffffll);
  __syncthreads();

  // a row's sequence is marked at the nearest marked row at or in front of it: a running maximum of marked places
  int place = m_seq[t] >= 0 ? t : -1;
  const int lane = t & 63, wave = t >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(place, d);
    if (lane >= d) place = up > place ? up : place;
  }
  if (lane == 63) wave_top[wave] = place;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < PL_THREADS / 64; w++) place = (w < wave && wave_top[w] > place) ? wave_top[w] : place;

  const long long row = (long long)row0 + t;
  if (row >= row1) return;
  int seq = -1, pos = 0;
  long long slot = -1;
  // rows behind the last sequence's are padding; `rows_before` is past them in every workgroup that has any
  if (place >= 0 && row < rows_before) {
    seq = m_seq[place];
    const long long at = (long long)m_ctx[place] + m_skip[place] + (t - place);
    pos = (int)(at < 0x7fffffffll ? at : 0x7fffffffll);
    const long long pidx = at >> page_bits;
    if (pidx < max_pages) {
      int* entry = table + (size_t)seq * max_pages + pidx;
      const int have = (int)(((long long)m_ctx[place] + page - 1) >> page_bits);
      int id;
      if (pidx >= have) {
        const long long f = m_first[place] + pidx;
        id = f < num_free ? free_pages[f] : -1;
        if ((at & (page - 1)) == 0) *entry = id;
      } else {
        id = *entry;
      }
      if (id >= 0) slot = ((long long)id << page_bits) + (at & (page - 1));
    }
  }
  positions[row] = pos;
  seq_ids[row] = seq;
  slots[row] = slot;
}

}  // namespace mi355

using namespace mi355;

extern "C" int mi355_paged_batch_layout(int32_t* block_table, const int32_t* context_lens, const int32_t* new_lens,
                                        const int32_t* free_pages, int64_t num_free, int64_t num_seqs,
                                        int64_t max_pages_per_seq, int64_t page_size, int64_t num_tokens, int32_t* seq_lens,
                                        int32_t* cu_new, int32_t* positions, int32_t* seq_ids, int64_t* slots,
                                        int32_t* pages_needed, void* stream) {
  const char* fn = "paged_batch_layout";
  if (!block_table || !context_lens || !new_lens || (!free_pages && num_free > 0) || !seq_lens || !cu_new || !positions ||
      !seq_ids || !slots || !pages_needed)
    return fail(-MI355_E_NULL, "%s: null pointer", fn);
  int page_bits = -1;
  for (int b = 4; b <= 8; b++)
    if (page_size == (1ll << b)) page_bits = b;
  if (page_bits < 0) return fail(-MI355_E_SHAPE, "%s: page size %lld not supported (16, 32, 64, 128 or 256)", fn, (long long)page_size);
  if (num_seqs <= 0 || num_seqs > 65535 || max_pages_per_seq <= 0 || max_pages_per_seq > (1 << 22) || num_tokens <= 0 ||
      num_tokens > (1 << 30) || num_free < 0 || num_free > (1 << 30))
    return fail(-MI355_E_SHAPE, "%s: bad sizes seqs=%lld max_pages=%lld tokens=%lld free=%lld", fn, (long long)num_seqs,
                (long long)max_pages_per_seq, (long long)num_tokens, (long long)num_free);
  // the first seven are written
  const Extent all[10] = {{block_table, num_seqs * max_pages_per_seq * 4}, {seq_lens, num_seqs * 4}, {cu_new, (num_seqs + 1) * 4}, {positions, num_tokens * 4},
                          {seq_ids, num_tokens * 4}, {slots, num_tokens * 8}, {pages_needed, 4}, {context_lens, num_seqs * 4}, {new_lens, num_seqs * 4},
                          {free_pages, num_free * 4}};
  for (int i = 0; i < 7; i++)
    for (int j = i + 1; j < 10; j++)
      if (overlap(all[i], all[j])) return fail(-MI355_E_OVERLAP, "%s: block_table and the outputs must not share memory with each other or with an input", fn);
  dim3 grid((unsigned)((num_tokens + PL_ROWS - 1) / PL_ROWS)), block(PL_THREADS);
  hipLaunchKernelGGL(paged_layout_kernel, grid, block, 0, reinterpret_cast<hipStream_t>(stream), block_table, context_lens,
                     new_lens, free_pages, (int)num_free, (int)num_seqs, (int)max_pages_per_seq, page_bits, (int)num_tokens,
                     seq_lens, cu_new, positions, seq_ids, reinterpret_cast<long long*>(slots), pages_needed);
  return check_launch("paged_layout_kernel", grid, block, 0);
}
