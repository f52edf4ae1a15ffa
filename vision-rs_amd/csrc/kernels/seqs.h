// Packed sequences on the device: where a sequence's queries and keys lie.
#pragma once
#include "common.h"

struct SeqSpan {
  int q0, q_len;      // rows of the queries
  int64_t k0;         // row of the first key
  int k_len;
  int k_lim;          // keys that lie inside the buffer (<= k_len)
};

// The last sequence whose first row is at or before `row` (sequences without
// rows are passed over), by a 64-way search: lane i probes one place, so n
// sequences cost log64(n) dependent loads.  start(i): first row (or tile) of
// sequence i, not falling with i; start(0) <= row.
template <typename F>
__device__ __forceinline__ int find_seq(int n, int row, F start) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 63) >> 6;
    const int i = lane * step;
    const uint64_t le = __ballot(i < len && start(lo + i) <= row);
    const int hit = le ? 63 - __builtin_clzll(le) : 0;
    lo += hit * step;
    len = min(step, len - hit * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Sequence i, cut to the buffers.
__device__ __forceinline__ SeqSpan seq_span(const vrs_seq_args& s, int i) {
  SeqSpan p;
  p.q0 = min(max(s.q_start[i], 0), s.q_rows);
  p.q_len = min(max(s.q_start[i + 1], p.q0), s.q_rows) - p.q0;
  p.k0 = s.k_start ? s.k_start[i] : p.q0;
  p.k_len = s.k_len ? max(s.k_len[i], 0) : p.q_len;
  p.k_lim = p.k0 < 0 || p.k0 >= s.k_rows ? 0 : (int)min((int64_t)p.k_len, s.k_rows - p.k0);
  return p;
}
