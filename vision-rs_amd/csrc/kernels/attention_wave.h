// What a wave of the attention kernels does: tiles of 32 queries x 32 keys on the
// matrix cores, softmax weights against a running reference, where rows and keys
// of a batch lie.
#pragma once
#include <type_traits>

#include "seqs.h"

namespace {
constexpr float kTau = 8.f;       // log2 units

typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2_t read_tr16(const bf16_t* p) {
  const v4i16_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16_t*)(p));
  return __builtin_bit_cast(u32x2_t, r);
}
// x combined with lane ^ 32's (v_permlane32_swap: the pair in either order, so symmetric uses only)
__device__ __forceinline__ float max32(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum32(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A query's weights are p = 2^(s c - R), one FMA and one v_exp, against a reference R that follows its
// running maximum m: R = m c rounded to float32, and every later factor is taken from that R, so its
// rounding weighs all keys alike.  Far from zero it could leave the range of 2^x: from |m c| = 2^30 on a
// power of two w >= c stands for c, whose products are exact.  Distinct scores are 2^6 log2 units apart
// there, so that the lower one weighs nothing on either.
constexpr float kFar = 1073741824.f;
constexpr float kNone = -3.40282347e38f;     // R before the first key: 2^(kNone - R) is 0, and so is p of a score -inf
struct Log2 {
  float c, w;
  __device__ __forceinline__ explicit Log2(float c_)
      : c(c_), w(__uint_as_float((__float_as_uint(c_) + 0x7fffffu) & 0x7f800000u)) {}
  static __device__ __forceinline__ bool far(float R) { return !(fabsf(R) < kFar); }
  __device__ __forceinline__ float unit(float R) const { return far(R) ? w : c; }
  __device__ __forceinline__ float reference(float m) const {
    const float R = m * c;
    return far(R) ? m * w : R;
  }
  // what weights on `from` are multiplied by on `to`
  __device__ __forceinline__ float factor(float from, float to) const {
#pragma clang fp contract(off)       // the references are rounded already
    float e = from - to;
    if (far(from) != far(to)) {      // the far one's m c, whole
      const float per_w = __uint_as_float(0x7f000000u - __float_as_uint(w));     // 1 / w
      e = far(from) ? __builtin_fmaf(from * per_w, c, -to) : -__builtin_fmaf(to * per_w, c, -from);
    }
    return __builtin_amdgcn_exp2f(e);
  }
};

// 1 / l; where no key weighs anything, 0 for a query that sees none and NaN for one all of whose keys
// score -inf.
__device__ __forceinline__ float share(float l, int keys) { return l == 0.f ? (keys > 0 ? NAN : 0.f) : 1.f / l; }

// A buffer resource in scalar registers, for load_lds.
__device__ __forceinline__ i32x4_hw lds_rsrc(const void* base, int bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  return (i32x4_hw){__builtin_amdgcn_readfirstlane((int)(uint32_t)b), __builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32) & 0xffff),
                    __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}

// Layout of a K or V tile in LDS: rows of D elements, 16-byte chunks XORed
// with bits of the row so that one instruction's lanes meet distinct banks
// (64 banks of 4 bytes): K's 16-byte reads take 16 rows at one chunk; V's
// transposed reads (bfloat16) 4 rows x 64 bytes, its float32 reads 128 bytes
// of rows r and r + 4.
template <typename T, int D>
struct Lds {
  static constexpr int CH = D * (int)sizeof(T) / 16;    // chunks of a row
  static __device__ __forceinline__ int kswz(int row) { return CH == 8 ? (row >> 1) & 7 : row & 15; }
  static __device__ __forceinline__ int vswz(int row) {
    if constexpr (sizeof(T) == 4) return ((row >> 2) & 1) << 3;
    else return CH == 8 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
  }
};

// Infinities and NaN of a 16-byte chunk become 0; whether there were any.
template <typename T>
__device__ __forceinline__ bool clean(u32x4_t& u) {
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool hi = (u[j] & 0x7f800000u) == 0x7f800000u;
    const bool lo = sizeof(T) == 2 && (u[j] & 0x7f80u) == 0x7f80u;
    bad |= hi || lo;
    u[j] &= sizeof(T) == 4 ? (hi ? 0u : ~0u) : (hi ? 0u : 0xffff0000u) | (lo ? 0u : 0xffffu);
  }
  return bad;
}

// One wave's QT tiles of 32 queries.
template <typename T, int D, int QT>
struct Wave {
  using E = Elt<T>;
  using G = typename E::group;
  static constexpr int PER = 16 / (int)sizeof(T);   // elements of a chunk
  G qf[QT][D / 16];
  f32x16_t o[QT][D / 32];
  float R[QT], l[QT];   // reference (see Log2) and this lane's share of the sum
  float unit[QT];       // c or w, as R has it (8192 causal queries: 503 us, 507 where each tile asks R)
  int lim[QT];          // keys that the lane's query sees
  int l32, hh;

  __device__ __forceinline__ void init(const Log2& u) {
    l32 = threadIdx.x & 31;
    hh = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      R[q] = kNone;
      unit[q] = u.w;
      l[q] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[q][t][r] = 0.f;
    }
  }
  // Q^T operand: 8 elements at s * 16 + hh * 8 of the lane's query
  __device__ __forceinline__ void load_q(int t, const T* q, int dim, bool ok) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const int d = s * 16 + hh * 8;
      qf[t][s] = ok && d < dim ? E::load(q + d) : E::zero();
    }
  }
  // register r of an S^T accumulator: key of the 32
  __device__ __forceinline__ int key_of(int r) const { return (r >> 2) * 8 + hh * 4 + (r & 3); }

  // scores of keys from lim on become -inf
  __device__ __forceinline__ void mask(int q, f32x16_t& s, int kc) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = kc + key_of(r) < lim[q] ? s[r] : -INFINITY;
  }
  static __device__ __forceinline__ float top(const f32x16_t& s) {
    float t = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, s[r]);
    return max32(t);
  }
  // the references follow the tile maxima t where one is exceeded by more than 2^kTau
  __device__ __forceinline__ void follow(const float (&t)[QT], const Log2& u) {
    bool over = false;
#pragma unroll
    for (int q = 0; q < QT; ++q) over |= __builtin_fmaf(t[q], unit[q], -R[q]) > kTau;
    if (__any(over)) {
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        const float to = __builtin_fmaf(t[q], unit[q], -R[q]) > 0.f ? u.reference(t[q]) : R[q];
        const float alpha = u.factor(R[q], to);
        R[q] = to;
        unit[q] = u.unit(to);
        l[q] *= alpha;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) o[q][d] *= alpha;
      }
    }
  }
  // scores -> probabilities: packed pairs (bfloat16, l summing the rounded ones) or float32
  struct P { uint32_t u[sizeof(T) == 2 ? 8 : 16]; };
  __device__ __forceinline__ P probs(int q, const f32x16_t& s, const Log2& u) {
    P p;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p.u[i] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], unit[q], -R[q])),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], unit[q], -R[q])));
        l[q] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v_t, p.u[i]),
                                               __builtin_bit_cast(bf16x2v_t, 0x3f803f80u), l[q], false);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], unit[q], -R[q]));
        p.u[r] = __float_as_uint(e);
        l[q] += e;
      }
    }
    return p;
  }

  // S^T of the 32 keys from `row` of a K tile in LDS
  __device__ __forceinline__ void scores(const T* sK, int row, f32x16_t (&s)[QT]) const {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[q][r] = 0.f;
    const int key = row + l32, z = Lds<T, D>::kswz(key);
    const T* base = sK + key * D;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      G kf;
      if constexpr (sizeof(T) == 2) {
        kf.v = *reinterpret_cast<const u32x4_t*>(base + ((2 * i + hh) ^ z) * PER);
      } else {
        kf.lo = *reinterpret_cast<const u32x4_t*>(base + ((4 * i + 2 * hh) ^ z) * PER);
        kf.hi = *reinterpret_cast<const u32x4_t*>(base + ((4 * i + 2 * hh + 1) ^ z) * PER);
      }
#pragma unroll
      for (int q = 0; q < QT; ++q) s[q] = mfma32_k16(kf, qf[q][i], s[q]);
    }
  }

  // This lane's V^T operand (bfloat16) for the 16 keys from `row`, channels d * 32 + 0..31
  __device__ __forceinline__ G vt(const T* sV, int row, int d) const {
    const int gi = threadIdx.x & 15;
    const int key = row + 4 * hh + (gi >> 2), vd = ((threadIdx.x >> 4) & 1) * 16 + 4 * (gi & 3);
    const int at = (((d * 32 + vd) >> 3) ^ Lds<T, D>::vswz(key)) * PER + (vd & 7);
    const u32x2_t lo = read_tr16(sV + key * D + at), hi = read_tr16(sV + (key + 8) * D + at);
    G vf;
    vf.v = (u32x4_t){lo[0], lo[1], hi[0], hi[1]};
    return vf;
  }
  // this lane's V^T value (float32) for register r's key of the 32 from `row`
  __device__ __forceinline__ float v1(const T* sV, int row, int r, int d) const {
    const int key = row + key_of(r), e = d * 32 + l32;
    return sV[key * D + (((e >> 2) ^ Lds<T, D>::vswz(key)) << 2) + (e & 3)];
  }

  // O^T += V^T P^T over the 32 keys from `row` of a V tile
  __device__ __forceinline__ void pv(const T* sV, int row, const P (&p)[QT]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const G vf = vt(sV, row + ks * 16, d);
#pragma unroll
          for (int q = 0; q < QT; ++q) {
            G pf;
            pf.v = (u32x4_t){p[q].u[4 * ks], p[q].u[4 * ks + 1], p[q].u[4 * ks + 2], p[q].u[4 * ks + 3]};
            o[q][d] = mfma32_k16(vf, pf, o[q][d]);
          }
        }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const float v = v1(sV, row, r, d);
#pragma unroll
          for (int q = 0; q < QT; ++q)
            o[q][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, __uint_as_float(p[q].u[r]), o[q][d], 0, 0, 0);
        }
    }
  }

  // Adds what the infinities and NaN among the 32 keys from kc (rows of v, n of them, dim elements)
  // give the queries that see them: for each sign, indicators of such values times indicators of
  // seen keys.  A NaN counts as an infinity of either sign (inf - inf).  Reads memory again: rare,
  // so small code rather than fast.
  __device__ __forceinline__ void add_specials(const T* v, int64_t ld, int n, int dim, int kc) {
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
#pragma unroll 1
        for (int sign = 0; sign < 2; ++sign) {
          const float inf = sign ? -INFINITY : INFINITY;
          f32x16_t count;
#pragma unroll
          for (int r = 0; r < 16; ++r) count[r] = 0.f;
#pragma unroll 1
          for (int r = 0; r < 16; ++r) {
            const int key = key_of(r), e = d * 32 + l32;
            const float x = key < n && e < dim ? E::to_f(v[key * ld + e]) : 0.f;
            count = __builtin_amdgcn_mfma_f32_32x32x2f32(x != x || x == inf ? 1.f : 0.f, kc + key < lim[q] ? 1.f : 0.f,
                                                         count, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) o[q][d][r] += count[r] > 0.f ? inf : 0.f;
        }
      }
  }

  // O / l of the lane's query to `out` (element type), `dim` elements
  __device__ __forceinline__ void store(int q, T* out, int dim, bool ok) const {
    const float lt = sum32(l[q]);
    const float inv = share(lt, lim[q]);
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int e = d * 32 + g * 8 + hh * 4;
          const f32x4_t v = {o[q][d][4 * g] * inv, o[q][d][4 * g + 1] * inv, o[q][d][4 * g + 2] * inv, o[q][d][4 * g + 3] * inv};
          if (ok && e < dim) *reinterpret_cast<f32x4_t*>(out + e) = v;
        }
      } else {
        // two quads of 4: the halves swapped so that each lane has 8 elements in a row
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          u32x2_t a = {pack_bf16x2(o[q][d][4 * g] * inv, o[q][d][4 * g + 1] * inv),
                       pack_bf16x2(o[q][d][4 * g + 2] * inv, o[q][d][4 * g + 3] * inv)};
          u32x2_t b = {pack_bf16x2(o[q][d][4 * g + 4] * inv, o[q][d][4 * g + 5] * inv),
                       pack_bf16x2(o[q][d][4 * g + 6] * inv, o[q][d][4 * g + 7] * inv)};
          const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
          const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
          const int e = d * 32 + g * 8 + hh * 8;
          if (ok && e < dim) *reinterpret_cast<u32x4_t*>(out + e) = (u32x4_t){x[0], y[0], x[1], y[1]};
        }
      }
    }
  }

  // adds parts of a workspace, `step` (row, head) apart, to the query's O, reference and sum
  __device__ __forceinline__ void take_parts(int q, const float* po, const float2* prl, int64_t step, int parts, int dim,
                                             const Log2& u) {
    float mx = R[q];
#pragma unroll 4
    for (int i = 0; i < parts; ++i) mx = fmaxf(mx, prl[i * step].x);
    const float mine = u.factor(R[q], mx);
    R[q] = mx;
    unit[q] = u.unit(mx);
    l[q] *= mine;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) o[q][d] *= mine;
#pragma unroll 1
    for (int i = 0; i < parts; ++i) {
      const float2 rl = prl[i * step];
      const float f = u.factor(rl.x, mx);
      if (hh == 0) l[q] += f * rl.y;         // (the halves of the wave add up their sums)
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int e = d * 32 + g * 8 + hh * 4;
          f32x4_t v = {0.f, 0.f, 0.f, 0.f};
          if (e < dim) v = *reinterpret_cast<const f32x4_t*>(po + i * step * dim + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) o[q][d][4 * g + k] += f * v[k];
        }
    }
  }

  // the unfinished query to a workspace: O (float32), reference, sum
  __device__ __forceinline__ void store_part(int q, float* po, float2* prl, int dim, bool ok) const {
    const float lt = sum32(l[q]);
    if (ok && hh == 0) *prl = make_float2(R[q], lt);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = d * 32 + g * 8 + hh * 4;
        const f32x4_t v = {o[q][d][4 * g], o[q][d][4 * g + 1], o[q][d][4 * g + 2], o[q][d][4 * g + 3]};
        if (ok && e < dim) *reinterpret_cast<f32x4_t*>(po + e) = v;
      }
  }
};

// Keys of a sequence that a query at place j of q_len sees.
__device__ __forceinline__ int visible(const SeqSpan& s, int j, int causal) {
  const int64_t own = (int64_t)s.k_len - s.q_len + j + 1;
  return (int)max(0l, causal ? min((int64_t)s.k_lim, own) : (int64_t)s.k_lim);
}
// Keys [kb, ke) of part `i` of `parts` of `keys` keys: equal whole tiles of `unit`.
__device__ __forceinline__ void part_of(int keys, int i, int parts, int unit, int& kb, int& ke) {
  const int tiles = (keys + unit - 1) / unit;
  kb = (int)((int64_t)tiles * i / parts) * unit;
  ke = min(keys, (int)((int64_t)tiles * (i + 1) / parts) * unit);
}

// Lane i's sequence, without another trip to memory.
__device__ __forceinline__ SeqSpan span_of_lane(const SeqSpan& s, int i) {
  SeqSpan p;
  p.q0 = __builtin_amdgcn_readlane(s.q0, i);
  p.q_len = __builtin_amdgcn_readlane(s.q_len, i);
  p.k0 = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(s.k0 >> 32), i) << 32) |
                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)s.k0, i));
  p.k_len = __builtin_amdgcn_readlane(s.k_len, i);
  p.k_lim = __builtin_amdgcn_readlane(s.k_lim, i);
  return p;
}
// Sum of x (or with ONES their number) over the lanes whose sequence comes
// before this lane's: those with more keys, or as many and a smaller number
// (from 2^25 keys on, as many).  Lanes without a sequence: keys -1.
template <bool ONES>
__device__ __forceinline__ int sum_before(int n, int keys, int x) {
  const int lane = threadIdx.x & 63;
  if (__ballot(lane < n && keys != __builtin_amdgcn_readfirstlane(keys)) == 0) {      // all alike: a prefix sum
    if constexpr (ONES) return lane;
    int sum = lane < n ? x : 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(sum, m);
      sum += lane >= m ? o : 0;
    }
    return sum - (lane < n ? x : 0);
  }
  // one number that orders both, and constant lanes: 64 sequences in about 1 us (3.5 in a plain loop)
  const int order = keys < 0 ? -1 : min(keys, (1 << 25) - 1) << 6 | (63 - lane);
  int before = 0;
#pragma unroll
  for (int c = 0; c < 64; c += 16) {
    if (c >= n) break;
#pragma unroll
    for (int k = c; k < c + 16; ++k) {
      const int kx = ONES ? 1 : __builtin_amdgcn_readlane(x, k);
      before += __builtin_amdgcn_readlane(order, k) > order ? kx : 0;
    }
  }
  return before;
}
// The sequences of a batch, for ranked_seq and place_tile.
struct Sequences {
  const vrs_seq_args& s;
  __device__ __forceinline__ int n() const { return s.n; }
  __device__ __forceinline__ SeqSpan span(int i) const { return seq_span(s, i); }
  __device__ __forceinline__ int row0(int i) const { return min(max(s.q_start[i], 0), s.q_rows); }
};
// The r-th sequence by number of keys, the most first (over 64: the r-th).
template <typename S>
__device__ __forceinline__ SeqSpan ranked_seq(const S& s, int r) {
  if (s.n() == 1 || s.n() > 64) return s.span(r);
  const int lane = threadIdx.x & 63;
  const SeqSpan sp = s.span(min(lane, s.n() - 1));
  const int rank = sum_before<true>(s.n(), lane < s.n() ? sp.k_len : -1, 1);
  return span_of_lane(sp, __builtin_ctzll(__ballot(lane < s.n() && rank == r)));
}
// Place of a row tile: its sequence, and which of its tiles (of BM rows; a
// query has `group` rows, one for each head of a key head).
struct TilePlace { SeqSpan sp; int tile; };
// Up to 64 sequences: those with the most keys first, so that the last
// workgroups to run are short ones; lane i holds sequence i, and its first id is
// the sum of the tiles of those before it.  More: in order, sequence i's ids
// from floor(first row / BM) + i, enough for each whatever the lengths.
// tile < 0: the id is none's.
template <int BM, typename S>
__device__ __forceinline__ TilePlace place_tile(const S& s, int group, int id) {
  if (s.n() <= 64) {
    const int lane = threadIdx.x & 63;
    const SeqSpan sp = s.span(min(lane, s.n() - 1));
    const int tiles = (int)(((int64_t)sp.q_len * group + BM - 1) / BM);
    const int before = sum_before<false>(s.n(), lane < s.n() ? sp.k_len : -1, tiles);
    const uint64_t hit = __ballot(id >= before && id < before + tiles && lane < s.n());
    const int at = hit ? __builtin_ctzll(hit) : 0;
    return {span_of_lane(sp, at), hit ? id - __builtin_amdgcn_readlane(before, at) : -1};
  }
  auto first = [&](int i) { return (int)((int64_t)s.row0(i) * group / BM) + i; };
  if (id < first(0)) return {SeqSpan{}, -1};
  const int sq = find_seq(s.n(), id, first);
  return {s.span(sq), id - first(sq)};
}

}  // namespace
