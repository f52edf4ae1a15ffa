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

// The group of the rows from q0 on, 64 probes at a time (uniform); q_len 0: none.
__device__ __forceinline__ SeqSpan group_of(const Groups& g, int q0) {
  SeqSpan s = {};
  if (g.n() == 0 || q0 < g.row0(0)) return s;
  s = g.span(find_seq(g.n(), q0, [&](int i) { return g.row0(i); }));
  if (q0 >= s.q0 + s.q_len) s = {};
  return s;
}
// Parts that a prefix of `keys` keys has: as the host counts on, of part_len each.
__device__ __forceinline__ int parts_of(const vrs_prefix_args& p, int keys) {
  return min(p.pre_parts, max(1, (int)(((int64_t)keys + p.part_len - 1) / p.part_len)));
}

// One launch for prefixes and own keys, all parts going to the workspace and to the join, or, where the own keys'
// rows are many (their parts would be most of the traffic), one for each, the second finishing what the first left
// (24 questions of 30 .. 200 tokens about 9000 keys: 505 + 33 us, 540 + 39 with the own keys in the first launch).
template <typename F>
__device__ __forceinline__ void job_of(const vrs_prefix_args& p, bool pre, int id, F place) {
  const vrs_attention_args& a = p.a;
  const int parts = pre ? p.pre_parts : p.own_parts;
  const int hk = id % a.kv, rest = id / a.kv, part = rest % parts;
  AttentionJob job = {};
  if (!place(rest / parts, job)) return;
  job.hk = hk;
  job.part = part;
  job.parts = parts;
  if (pre) {
    job.out_part = part;
    job.part_len = p.part_len;
    if (part >= parts_of(p, job.sp.k_lim)) job.sp.q_len = 0;         // no such part
  } else {
    job.out_part = p.pre_parts + part;
    job.causal = a.causal;
    if (p.finish) {
      job.direct = true;
      const SeqSpan g = group_of(Groups{p}, job.sp.q0);
      job.joined = g.q_len ? parts_of(p, g.k_lim) : 0;
      job.joined_keys = g.q_len ? g.k_lim : 0;
    }
  }
  if (job.sp.q_len > 0) place(-1, job);
}
template <typename T, int D, bool PRE>
__device__ __forceinline__ void prompt_job(const vrs_prefix_args& p, int id0) {
  job_of(p, PRE, id0, [&](int id, AttentionJob& job) {
    if (id < 0) {
      prompt_body<T, D, 32, 1, 4>(p.a, job);
      return true;
    }
    TilePlace at;
    if constexpr (PRE) at = place_tile<128>(Groups{p}, p.a.heads / p.a.kv, id);
    else at = place_tile<128>(Sequences{p.a.s}, p.a.heads / p.a.kv, id);
    job.sp = at.sp;
    job.tile = at.tile;
    return at.tile >= 0;
  });
}
template <typename T, int D, bool SHARED>
__device__ __forceinline__ void few_job(const vrs_prefix_args& p, bool pre, int id0) {
  const int tiles = pre ? p.pre_rows : p.own_rows;
  if ((int)blockIdx.y >= tiles) return;
  job_of(p, pre, id0, [&](int id, AttentionJob& job) {
    if (id < 0) {
      few_body<T, D, 4, SHARED>(p.a, job);
      return true;
    }
    if (pre) job.sp = ranked_seq(Groups{p}, id);
    else job.sp = ranked_seq(Sequences{p.a.s}, id);
    job.tile = blockIdx.y;
    job.step = tiles;
    return true;
  });
}
template <typename T, int D>
__device__ __forceinline__ void few_kernel(const vrs_prefix_args& p) {
  const bool pre = (int)blockIdx.x < p.pre_blocks;
  few_job<T, D, false>(p, pre, blockIdx.x - (pre ? 0 : p.pre_blocks));
}
// Many rows to a prefix, few to a sequence: both kinds in one launch, the few first, which are bound by memory and
// unequal (64 tokens on four prefixes of 1500 .. 6000 keys, 20 .. 700 own, 32 heads on 8 of 128: 40 us, 42 with
// the prefixes first, 28 + 18 in two launches; the join takes 7).
template <typename T, int D>
__device__ __forceinline__ void mixed_kernel(const vrs_prefix_args& p) {
  const int own = gridDim.x - p.pre_blocks;
  if ((int)blockIdx.x < own) few_job<T, D, true>(p, false, blockIdx.x);
  else if (blockIdx.y == 0) prompt_job<T, D, true>(p, blockIdx.x - own);
}

// Joins the parts: a workgroup takes a row, a thread 4 elements of a head.
template <typename T>
__device__ __forceinline__ void join_body(const vrs_prefix_args& p) {
  const vrs_attention_args& a = p.a;
  const int row = blockIdx.x;
  if (row < a.s.q_start[0]) return;
  const SeqSpan sp = seq_span(a.s, find_seq(a.s.n, row, [&](int i) { return a.s.q_start[i]; }));
  if (row < sp.q0 || row >= sp.q0 + sp.q_len) return;
  const int per = a.dim / 4, t = blockIdx.y * 256 + threadIdx.x, h = t / per, e = (t - h * per) * 4;
  const SeqSpan g = group_of(Groups{p}, sp.q0);      // (by all lanes of a wave)
  if (h >= a.heads) return;
  const int pre = g.q_len ? parts_of(p, g.k_lim) : 0, parts = pre + p.own_parts;
  const int keys = (int)min((int64_t)visible(sp, row - sp.q0, a.causal) + (g.q_len ? g.k_lim : 0), (int64_t)0x7fffffff);
  const int64_t step = (int64_t)a.s.q_rows * a.heads, id = (int64_t)row * a.heads + h;
  const Log2 u(a.c);
  constexpr int N = 8;                         // parts on their way at once
  float mx = kNone, l = 0.f;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < parts; i0 += N) {
    float2 rl[N];
    f32x4_t o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i0 + i >= parts) continue;
      const int part = i0 + i < pre ? i0 + i : p.pre_parts + i0 + i - pre;
      rl[i] = a.part_rl[part * step + id];
      o[i] = *reinterpret_cast<const f32x4_t*>(a.part_o + (part * step + id) * a.dim + e);
    }
    float to = mx;
#pragma unroll
    for (int i = 0; i < N; ++i) to = i0 + i < parts ? fmaxf(to, rl[i].x) : to;
    const float old = u.factor(mx, to);
    mx = to;
    l *= old;
    v *= old;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i0 + i >= parts) continue;
      const float f = u.factor(rl[i].x, mx);   // (no key seen: l, O are 0)
      l += f * rl[i].y;
      v += f * o[i];
    }
  }
  v *= share(l, keys);
  T* out = static_cast<T*>(a.out) + (int64_t)row * a.o_ld + (int64_t)h * a.o_hd + e;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(out) = v;
  else *reinterpret_cast<u32x2_t*>(out) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
}  // namespace

#define VRS_PREFIX(TN, T, D, WPS)                                                                                             \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_prompt_##TN##_d##D(vrs_prefix_args p) { prompt_job<T, D, true>(p, blockIdx.x); } \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_own_##TN##_d##D(vrs_prefix_args p) { prompt_job<T, D, false>(p, blockIdx.x); }
#define VRS_PREFIX_FEW(TN, T, D, WPS)                                                                                         \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_few_##TN##_d##D(vrs_prefix_args p) { few_kernel<T, D>(p); } \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_prefix_mixed_##TN##_d##D(vrs_prefix_args p) { mixed_kernel<T, D>(p); }
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
