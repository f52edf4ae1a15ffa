// Attention over packed sequences and over a cache, for gfx950:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys j < lim_i of the query's sequence (causal: those at or before
// its own place; else all), with grouped heads (heads / kv_heads queries to a
// key head) and head sizes up to 64 or 128 (shorter ones padded by loads that
// read zeros).
//
// Both kernels work in wave tiles of 32 queries x 32 keys:
//   S^T(keys x queries) = K Q^T     on 32x32 MFMA, K rows as A, Q^T as B
//   p = 2^(s c - R)                 c = scale log2 e, R near m c (Log2)
//   O^T(d x queries) += V^T P^T     the accumulator of S^T is already P^T's
//                                   operand layout, V^T in the same key order
// A lane holds 16 keys of one query, so the row maximum and sum need one
// exchange with lane ^ 32 and the rescale of O is a lane's own factor.  The
// running maximum moves only where a tile exceeds it by over 2^8 (p <= 256
// meanwhile), so rescales of O are rare.  Scores, p, m, l and O are float32;
// bfloat16 rounds p once, for the second product, and l sums the rounded p,
// so a dominant p's rounding cancels in O / l.
//
// Keys that a query must not see have p = 0, which hides any finite v; a v
// that is not finite would still make 0 * v a NaN.  So where a tile has masked
// keys, values that are not finite are staged as 0, and if there were any,
// products of indicators add them to the queries that see them
// (add_specials).  Keys behind a sequence's last are not read at all.
#include "attention_body.h"

namespace {
// Prompts: key heads innermost, so that workgroups dealt round the 8 XCDs give each XCD few heads' keys
// (one of 8, three of 12) and as many long tiles as any other.
template <typename T, int D, int KT, int QT, int NW>
__device__ __forceinline__ void prompt_kernel(const vrs_attention_args& a) {
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv;
  const int part = rest % a.parts;
  const TilePlace at = place_tile<32 * NW * QT>(Sequences{a.s}, a.heads / a.kv, rest / a.parts);
  if (at.tile < 0) return;
  prompt_body<T, D, KT, QT, NW>(a, {at.sp, hk, at.tile, 0, part, a.parts, part, a.causal, a.parts == 1, 0, 0, 0});
}
// Few queries: no two workgroups share keys: in the order of launch, round the XCDs, the sequences with
// the most keys first.
template <typename T, int D, int NW>
__device__ __forceinline__ void few_kernel(const vrs_attention_args& a) {
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv;
  const int part = rest % a.parts;
  few_body<T, D, NW>(a, {ranked_seq(Sequences{a.s}, rest / a.parts), hk, (int)blockIdx.y, (int)gridDim.y, part, a.parts, part,
                         a.causal, a.parts == 1, 0, 0, 0});
}

// ---------------------------------------------------------------------------
// Joins the parts of the keys: a thread takes 4 elements of one (row, head).
template <typename T>
__device__ __forceinline__ void join_body(const vrs_attention_args& a) {
  const int per = a.dim / 4;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t id = t / per;
  const int e = (int)(t - id * per) * 4;
  const int64_t row = id / a.heads;
  const int h = (int)(id - row * a.heads);
  if (row >= a.s.q_rows || row < a.s.q_start[0]) return;
  int sq = 0;
  for (int n = a.s.n; n > 1;) {          // the last sequence that starts at or before the row
    const int half = n / 2;
    if (a.s.q_start[sq + half] <= row) sq += half, n -= half;
    else n = half;
  }
  const SeqSpan sp = seq_span(a.s, sq);
  if (row < sp.q0 || row >= sp.q0 + sp.q_len) return;
  const int64_t step = (int64_t)a.s.q_rows * a.heads;
  const Log2 u(a.c);
  float mx = kNone;
#pragma unroll 4
  for (int p = 0; p < a.parts; ++p) mx = fmaxf(mx, a.part_rl[p * step + id].x);
  float l = 0.f;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < a.parts; ++p) {
    const float2 rl = a.part_rl[p * step + id];
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(a.part_o + (p * step + id) * a.dim + e);
    const float f = u.factor(rl.x, mx);          // (no key seen: l, O are 0)
    l += f * rl.y;
    v += f * o;
  }
  v *= share(l, visible(sp, (int)(row - sp.q0), a.causal));
  T* out = static_cast<T*>(a.out) + row * a.o_ld + h * a.o_hd + e;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(out) = v;
  else *reinterpret_cast<u32x2_t*>(out) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
}  // namespace

#define VRS_ATTENTION_PROMPT(TN, T, D, KT, QT, NW, WPS)                                                                      \
  extern "C" __global__ __launch_bounds__(64 * NW, WPS) void vrs_attention_prompt_##TN##_d##D##_q##QT##_w##NW(vrs_attention_args a) { \
    prompt_kernel<T, D, KT, QT, NW>(a);                                                                                         \
  }
#define VRS_ATTENTION_FEW(TN, T, D, NW, WPS)                                                                               \
  extern "C" __global__ __launch_bounds__(64 * NW, WPS) void vrs_attention_few_##TN##_d##D##_w##NW(vrs_attention_args a) { \
    few_kernel<T, D, NW>(a);                                                                                                 \
  }
VRS_ATTENTION_PROMPT(bf16, bf16_t, 64, 32, 1, 4, 4)
VRS_ATTENTION_PROMPT(bf16, bf16_t, 64, 64, 2, 4, 2)
VRS_ATTENTION_PROMPT(bf16, bf16_t, 128, 32, 1, 4, 2)
VRS_ATTENTION_PROMPT(bf16, bf16_t, 128, 64, 1, 8, 2)
VRS_ATTENTION_PROMPT(f32, float, 64, 32, 1, 4, 3)
VRS_ATTENTION_PROMPT(f32, float, 64, 32, 1, 8, 2)
VRS_ATTENTION_PROMPT(f32, float, 128, 32, 1, 4, 2)
VRS_ATTENTION_PROMPT(f32, float, 128, 32, 1, 8, 2)
VRS_ATTENTION_FEW(bf16, bf16_t, 64, 4, 2)
VRS_ATTENTION_FEW(bf16, bf16_t, 128, 4, 2)
VRS_ATTENTION_FEW(bf16, bf16_t, 64, 8, 2)
VRS_ATTENTION_FEW(bf16, bf16_t, 128, 8, 2)
VRS_ATTENTION_FEW(f32, float, 64, 4, 1)
VRS_ATTENTION_FEW(f32, float, 128, 4, 1)
extern "C" __global__ __launch_bounds__(256) void vrs_attention_join_bf16(vrs_attention_args a) { join_body<bf16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_attention_join_f32(vrs_attention_args a) { join_body<float>(a); }
