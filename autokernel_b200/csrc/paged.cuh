// The paged key/value cache shared by the append and attention kernels.
//
// N packed tokens of B sequences: tokens cu_q[b] .. cu_q[b + 1] - 1 are sequence b's new tokens
// (n_b of them), kv_lens[b] its keys with the new ones, so its token i sits at position
// kv_lens[b] - n_b + i.  Position p lies in slot p % S of page page_table[b][p / S]; a cache is
// [P, Hkv, S, D] given by element strides {page, head, slot} with D contiguous.
//
// The lists live on the device and no host code reads them, so the kernels clamp what they
// read: a token range is cut to [0, N), and a page is only followed when it lies in [0, P) and in
// the table's row.  A key that has no such page is a missing key; what that means for the
// result is each operator's rule.
#pragma once
#include "ak_common.cuh"

namespace ak {

struct PagedLists {
  const int32_t* page_table;  // [B, max_pages], row stride table_ld
  const int32_t* cu_q;        // [B + 1]
  const int32_t* kv_lens;     // [B]
  int64_t table_ld;
  int N, B;
  int max_pages, num_pages, page_size;
};

// Whether the rows of `inner` contiguous elements that n <= 3 strided dims name may share elements: an output
// of such a layout would be written by several threads at once.
inline bool may_overlap(const int64_t* sizes, const int64_t* strides, int n, int64_t inner) {
  int order[3], m = 0;
  for (int i = 0; i < n; ++i) {  // the dims of more than one element, by stride
    if (sizes[i] <= 1) continue;
    int at = m++;
    for (; at > 0 && strides[order[at - 1]] > strides[i]; --at) order[at] = order[at - 1];
    order[at] = i;
  }
  int64_t extent = inner;  // of what the dims so far span
  for (int k = 0; k < m; ++k) {
    if (strides[order[k]] < extent) return true;
    extent += (sizes[order[k]] - 1) * strides[order[k]];
  }
  return false;
}

struct SeqRange {
  int begin, n;    // first packed token, number of new tokens
  int kv_len;      // keys, the new tokens counted (may exceed what the table can name)
};

AK_D SeqRange seq_range(const PagedLists& l, int b) {
  SeqRange r;
  const int lo = min(max(__ldg(l.cu_q + b), 0), l.N);
  const int hi = min(max(__ldg(l.cu_q + b + 1), 0), l.N);
  r.begin = lo;
  r.n = max(hi - lo, 0);
  r.kv_len = max(__ldg(l.kv_lens + b), 0);
  return r;
}

// Page of page index i of sequence b, or -1 when the key has none.
AK_D int page_of(const PagedLists& l, int b, int i) {
  if ((unsigned)i >= (unsigned)l.max_pages) return -1;
  const int p = __ldg(l.page_table + (int64_t)b * l.table_ld + i);
  return (unsigned)p < (unsigned)l.num_pages ? p : -1;
}

// Sequence of packed token t for a whole warp: the last b with cu_q[b] <= t.  32 probes a round
// (two rounds up to 1024 sequences) instead of one dependent load per bit.  Returns B when t
// lies behind the last sequence, -1 when it lies before the first.
AK_D int seq_of_token_warp(const PagedLists& l, int t) {
  const int lane = threadIdx.x & 31;
  int lo = -1, hi = l.B + 1;  // cu_q[lo] <= t < cu_q[hi] with cu_q[-1] = -inf, cu_q[B+1] = +inf
  while (hi - lo > 1) {
    const int span = hi - lo, step = (span + 32) / 33;
    const int i = lo + (lane + 1) * step;
    const bool le = i < hi && __ldg(l.cu_q + i) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    lo += c * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace ak
