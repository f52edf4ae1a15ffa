// Attention of sequences that share a prefix, for gfx950:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys of the sequence's group (the prefix, all of which every query
// sees) and then the sequence's own.  The softmax over both runs is the joined one
// of each: a part of the keys leaves O, its reference R and its sum l, and
//   o = sum_p 2^(R_p - R) O_p / sum_p 2^(R_p - R) l_p.
// Queries of a group lie together, so that the group is one long sequence of
// queries to its prefix: the prefix is read for 32 or 128 rows at a time (a row is
// a query and head) instead of once for each sequence.
#include "attention_body.h"

namespace {

// Groups as sequences: the rows of all their sequences, the keys of the prefix.
struct Groups {
  const vrs_prefix_args& p;
  __device__ __forceinline__ int n() const { return p.groups; }
  __device__ __forceinline__ int seq0(int g) const { return min(max(p.first[g], 0), p.a.s.n); }
  __device__ __forceinline__ int row0(int g) const { return min(max(p.a.s.q_start[seq0(g)], 0), p.a.s.q_rows); }
  __device__ __forceinline__ SeqSpan span(int g) const {
    const vrs_seq_args& s = p.a.s;
    SeqSpan o;
    const int i1 = min(max(p.first[g + 1], seq0(g)), s.n);
    o.q0 = row0(g);
    o.q_len = min(max(s.q_start[i1], o.q0), s.q_rows) - o.q0;
    o.k0 = p.p_start[g];
    o.k_len = max(p.p_len[g], 0);
    o.k_lim = o.k0 < 0 || o.k0 >= s.k_rows ? 0 : (int)min((int64_t)o.k_len, s.k_rows - o.k0);
    return o;
  }
};

// Both kernels: the workgroups of the prefixes first, whose keys are the most.
template <typename T, int D>
__device__ __forceinline__ void prompt_kernel(const vrs_prefix_args& p) {
  const vrs_attention_args& a = p.a;
  const bool pre = (int)blockIdx.x < p.pre_blocks;
  const int id = blockIdx.x - (pre ? 0 : p.pre_blocks), parts = pre ? p.pre_parts : p.own_parts;
  const int hk = id % a.kv, rest = id / a.kv, part = rest % parts, group = a.heads / a.kv;
  TilePlace at;
  if (pre) at = place_tile<128>(Groups{p}, group, rest / parts);
  else at = place_tile<128>(Sequences{a.s}, group, rest / parts);
  if (at.tile < 0) return;
  prompt_body<T, D, 32, 1, 4>(a, {at.sp, hk, at.tile, 0, part, parts, pre ? part : p.pre_parts + part, pre ? 0 : a.causal, false});
}
template <typename T, int D>
__device__ __forceinline__ void few_kernel(const vrs_prefix_args& p) {
  const vrs_attention_args& a = p.a;
  const bool pre = (int)blockIdx.x < p.pre_blocks;
  const int id = blockIdx.x - (pre ? 0 : p.pre_blocks), parts = pre ? p.pre_parts : p.own_parts;
  const int tiles = pre ? p.pre_rows : p.own_rows;
  if ((int)blockIdx.y >= tiles) return;
  const int hk = id % a.kv, rest = id / a.kv, part = rest % parts;
  SeqSpan sp;
  if (pre) sp = ranked_seq(Groups{p}, rest / parts);
  else sp = ranked_seq(Sequences{a.s}, rest / parts);
  few_body<T, D, 4>(a, {sp, hk, (int)blockIdx.y, tiles, part, parts, pre ? part : p.pre_parts + part, pre ? 0 : a.causal, false});
}

// The last of n whose first row (or sequence) is at or before x.
template <typename F>
__device__ __forceinline__ int last_at(int n, int64_t x, F start) {
  int at = 0;
  while (n > 1) {
    const int half = n / 2;
    if (start(at + half) <= x) at += half, n -= half;
    else n = half;
  }
  return at;
}

// Joins the parts: a thread takes 4 elements of one (row, head).
template <typename T>
__device__ __forceinline__ void join_body(const vrs_prefix_args& p) {
  const vrs_attention_args& a = p.a;
  const int per = a.dim / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t id = t / per;
  const int e = (int)(t - id * per) * 4;
  const int64_t row = id / a.heads;
  const int h = (int)(id - row * a.heads);
  if (row >= a.s.q_rows || row < a.s.q_start[0]) return;
  const int sq = last_at(a.s.n, row, [&](int i) { return a.s.q_start[i]; });
  const SeqSpan sp = seq_span(a.s, sq);
  if (row < sp.q0 || row >= sp.q0 + sp.q_len) return;
  // the group, by its rows: where no prefix part wrote this row, there is none
  const Groups groups{p};
  int from = p.pre_parts, keys = visible(sp, (int)(row - sp.q0), a.causal);
  if (p.groups && row >= groups.row0(0)) {
    const SeqSpan g = groups.span(last_at(p.groups, row, [&](int i) { return groups.row0(i); }));
    if (row < g.q0 + g.q_len) from = 0, keys = (int)min((int64_t)keys + g.k_lim, (int64_t)0x7fffffff);
  }
  const int64_t step = (int64_t)a.s.q_rows * a.heads;
  const Log2 u(a.c);
  float mx = kNone;
#pragma unroll 4
  for (int i = from; i < a.parts; ++i) mx = fmaxf(mx, a.part_rl[i * step + id].x);
  float l = 0.f;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = from; i < a.parts; ++i) {
    const float2 rl = a.part_rl[i * step + id];
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(a.part_o + (i * step + id) * a.dim + e);
    const float f = u.factor(rl.x, mx);          // (no key seen: l, O are 0)
    l += f * rl.y;
    v += f * o;
  }
  v *= share(l, keys);
  T* out = static_cast<T*>(a.out) + row * a.o_ld + h * a.o_hd + e;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(out) = v;
  else *reinterpret_cast<u32x2_t*>(out) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
}  // namespace

#define VRS_PREFIX(TN, T, D, WPS)                                                                                             \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_prompt_##TN##_d##D(vrs_prefix_args p) { prompt_kernel<T, D>(p); }
#define VRS_PREFIX_FEW(TN, T, D, WPS)                                                                                         \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_few_##TN##_d##D(vrs_prefix_args p) { few_kernel<T, D>(p); }
VRS_PREFIX(bf16, bf16_t, 64, 4)
VRS_PREFIX(bf16, bf16_t, 128, 2)
VRS_PREFIX(f32, float, 64, 3)
VRS_PREFIX(f32, float, 128, 1)
VRS_PREFIX_FEW(bf16, bf16_t, 64, 2)
VRS_PREFIX_FEW(bf16, bf16_t, 128, 2)
VRS_PREFIX_FEW(f32, float, 64, 1)
VRS_PREFIX_FEW(f32, float, 128, 1)
extern "C" __global__ __launch_bounds__(256) void vrs_prefix_join_bf16(vrs_prefix_args p) { join_body<bf16_t>(p); }
extern "C" __global__ __launch_bounds__(256) void vrs_prefix_join_f32(vrs_prefix_args p) { join_body<float>(p); }
