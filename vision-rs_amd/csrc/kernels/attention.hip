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
// The r-th sequence by number of keys, the most first (over 64: the r-th).
__device__ __forceinline__ SeqSpan ranked_seq(const vrs_seq_args& s, int r) {
  if (s.n == 1 || s.n > 64) return seq_span(s, r);
  const int lane = threadIdx.x & 63;
  const SeqSpan sp = seq_span(s, min(lane, s.n - 1));
  const int rank = sum_before<true>(s.n, lane < s.n ? sp.k_len : -1, 1);
  return span_of_lane(sp, __builtin_ctzll(__ballot(lane < s.n && rank == r)));
}
// Place of a row tile: its sequence, and which of its tiles (of BM rows; a
// query has `group` rows, one for each head of a key head).
struct TilePlace { SeqSpan sp; int tile; };
// Up to 64 sequences: those with the most keys first, so that the last
// workgroups to run are short ones; lane i holds sequence i, and its first id is
// the sum of the tiles of those before it.  More: in order, sequence i's ids
// from floor(first row / BM) + i, enough for each whatever the lengths.
// tile < 0: the id is none's.
template <int BM>
__device__ __forceinline__ TilePlace place_tile(const vrs_seq_args& s, int group, int id) {
  if (s.n <= 64) {
    const int lane = threadIdx.x & 63;
    const SeqSpan sp = seq_span(s, min(lane, s.n - 1));
    const int tiles = (int)(((int64_t)sp.q_len * group + BM - 1) / BM);
    const int before = sum_before<false>(s.n, lane < s.n ? sp.k_len : -1, tiles);
    const uint64_t hit = __ballot(id >= before && id < before + tiles && lane < s.n);
    const int at = hit ? __builtin_ctzll(hit) : 0;
    return {span_of_lane(sp, at), hit ? id - __builtin_amdgcn_readlane(before, at) : -1};
  }
  auto first = [&](int i) { return (int)((int64_t)min(max(s.q_start[i], 0), s.q_rows) * group / BM) + i; };
  if (id < first(0)) return {SeqSpan{}, -1};
  const int sq = find_seq(s.n, id, first);
  return {seq_span(s, sq), id - first(sq)};
}

// ---------------------------------------------------------------------------
// Prompts: a workgroup of 4 waves takes 128 * QT rows, the queries of all heads
// of one key head (neighbouring rows share a query, so causal tiles waste
// little and the keys serve the whole group), a wave 32 * QT of them; K and V
// tiles of KT keys are shared through LDS.
//
// The loop is written as a software pipeline: the next 32 keys' scores are
// multiplied between these 32 keys' maximum and their exponentials, so that
// neither kind of instruction waits for the other's results.  Measured per 32
// keys x 32 queries and SIMD: 512 cycles of matrix instructions and 459 of
// vector ones in 1020 at D = 128, 256 and 475 in 713 at D = 64: close to their
// sums, so the waves of a SIMD hardly overlap one kind with the other, and
// neither unit is full (50 and 45 % at 128, 36 and 67 % at 64).
//
// LDS holds three tiles, filled by loads that go straight there: one barrier
// before tile i's last 32 keys (whose step reads tile i + 1's first scores)
// makes tile i + 1 visible and frees tile i - 1's place for tile i + 2, whose
// loads then have a whole tile's time.  Tiles that some row does not see whole
// take the general form of the step; the others three at a time, so that LDS
// addresses are constants.
//
// 8192 causal queries, 32 heads on 8 of 128: 500 .. 540 us queued (cards and
// their clock under this load differ), 1020 .. 1100 TFLOP/s; an 8192^3 product
// reaches 1110 .. 1160.  Traced one by one: 568 us at 1.86 GHz, 1.05 M cycles,
// rising to 670 as the clock falls to 1.52.  No LDS bank conflicts.  8 waves and
// 64-key tiles against 4 waves and 32: 516 us to 548.  At head sizes up to 64 the
// same exponentials serve half the products: 24 images of 196 .. 1600 patches,
// 12 heads: 120 .. 128 us, 700 TFLOP/s; four 4-wave workgroups on a CU with
// 32-key tiles against three with 64: 124 us to 130; two query tiles to a wave
// for the large (4096 x 32 heads: 148 us to 159).  Heads of 72 .. 120 run padded
// to 128 (64 sequences of 512, 16 heads: 64 113 us, 72 177, 80 180, 96 191, 128
// 207).  float32 is bound by its matrix instructions (64 cycles each).
template <typename T, int D, int KT, int QT, int NW>
__device__ __forceinline__ void prompt_body(const vrs_attention_args& a) {
  constexpr int NT = 64 * NW, BM = 32 * NW * QT, NS = KT / 32;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = KT * CH / NT;                 // chunks a thread stages of K, and of V
  constexpr int TILE = KT * D;
  __shared__ __attribute__((aligned(16))) T smem[3 * 2 * TILE];    // three times K, V
  __shared__ int odd_tile[3];     // first key of the tile that a buffer holds, if it had values not finite
  const int tid = threadIdx.x, wave = tid >> 6;
  // Key heads innermost, so that workgroups dealt round the 8 XCDs give each XCD
  // few heads' keys (one of 8, three of 12) and as many long tiles as any other.
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv;
  const int part = rest % a.parts;
  const int group = a.heads / a.kv;
  const TilePlace at = place_tile<BM>(a.s, group, rest / a.parts);
  if (at.tile < 0) return;
  const SeqSpan sp = at.sp;
  const int64_t rows = (int64_t)sp.q_len * group;
  const int tiles = (int)((rows + BM - 1) / BM);
  if (at.tile >= tiles) return;
  const int64_t r0 = (int64_t)(tiles - 1 - at.tile) * BM;     // late rows (causal: the most keys) first

  const Log2 u(a.c);
  Wave<T, D, QT> w;
  w.init(u);
  int64_t qrow[QT];
  int head[QT];
  bool ok[QT];
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    const int64_t r = r0 + wave * 32 * QT + q * 32 + w.l32;
    ok[q] = r < rows;
    const int j = (int)(min(r, rows - 1) / group);
    head[q] = hk * group + (int)(min(r, rows - 1) - (int64_t)j * group);
    qrow[q] = sp.q0 + j;
    w.lim[q] = visible(sp, j, a.causal);
    w.load_q(q, static_cast<const T*>(a.q) + qrow[q] * a.q_ld + head[q] * a.q_hd, a.dim, ok[q]);
  }
  int kb, ke;
  part_of(visible(sp, (int)((min(r0 + BM, rows) - 1) / group), a.causal), part, a.parts, KT, kb, ke);
  const int all = visible(sp, (int)(r0 / group), a.causal);   // keys that every row of the workgroup sees
  const int mine = __builtin_amdgcn_readlane(w.lim[QT - 1], 31);   // keys that some row of the wave sees

  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
  // A thread's chunks of a tile, straight to LDS: one instruction of a wave fills 1 KiB in lane
  // order, so the swizzle is in what each lane loads.  Elements past the head and keys past the
  // sequence's last are out of the buffer's range and fill in 0; such keys are masked besides.
  uint32_t ko[IT], vo[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int slot = (i * NW + wave) * 64 + (tid & 63), row = slot / CH, at = slot % CH;
    const int kc = (at ^ Lds<T, D>::kswz(row)) * PER, vc = (at ^ Lds<T, D>::vswz(row)) * PER;
    ko[i] = kc < a.dim ? (uint32_t)(row * (int)a.k_ld + kc) * (uint32_t)sizeof(T) : kOOB;
    vo[i] = vc < a.dim ? (uint32_t)(row * (int)a.v_ld + vc) * (uint32_t)sizeof(T) : kOOB;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem + wave * 1024);
  auto load = [&](int buf, int kc) {
    const int n = min(KT, sp.k_lim - kc);
    const i32x4_hw rk = lds_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
    const i32x4_hw rv = lds_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((n - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
    const uint32_t to = lds0 + buf * 2 * TILE * (uint32_t)sizeof(T);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_lds(rk, ko[i], to + i * NW * 1024);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_lds(rv, vo[i], to + TILE * (uint32_t)sizeof(T) + i * NW * 1024);
  };
  // V of a tile that some row does not see whole: values that are not finite become 0
  auto clean_tile = [&](int buf, int kc) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      u32x4_t* at = reinterpret_cast<u32x4_t*>(smem + (buf * 2 + 1) * TILE) + (i * NW + wave) * 64 + (tid & 63);
      u32x4_t u = *at;
      if (clean<T>(u)) {
        *at = u;
        bad = true;
      }
    }
    if (bad) odd_tile[buf] = kc;
  };
  if (kb < ke) {
    if (tid < 3) odd_tile[tid] = -1;
    load(0, kb);
    if (kb + KT < ke) {
      load(1, kb + KT);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * IT) : "memory");   // the first tile is there
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
    f32x16_t s[QT];
    float t[QT];
    int kc = kb;
    // maximum of 32 keys' scores, of which those a query does not see are masked first
    auto look = [&](bool masked, int key) {
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        if (masked) w.mask(q, s[q], key);
        t[q] = w.top(s[q]);
      }
    };
    w.scores(smem, 0, s);
    look(kb + 32 > all, kb);
    // TAIL: some row does not see the whole of this or the next tile, or no tile follows
    auto tile = [&](auto tail, int buf, bool more) {
      constexpr bool TAIL = decltype(tail)::value;
      const int nbuf = buf == 2 ? 0 : buf + 1;
      const T* sK = smem + buf * 2 * TILE;
      if (TAIL && kc + KT > all) clean_tile(buf, kc);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const bool last = n == NS - 1;
        const bool live = !TAIL || kc + n * 32 < mine;
        if (live) w.follow(t, u);
        if (last) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the next tile
        if (last || (TAIL && kc + KT > all)) __syncthreads();
        if (last && kc + 2 * KT < ke) load(buf == 0 ? 2 : buf - 1, kc + 2 * KT);
        f32x16_t s1[QT];
        const bool ahead = !TAIL || ((!last || more) && kc + (n + 1) * 32 < mine);
        __builtin_amdgcn_s_setprio(1);
        if (ahead) w.scores(last ? smem + nbuf * 2 * TILE : sK, last ? 0 : (n + 1) * 32, s1);
        if (live) {
          typename Wave<T, D, QT>::P p[QT];
#pragma unroll
          for (int q = 0; q < QT; ++q) p[q] = w.probs(q, s[q], u);
          w.pv(sK + TILE, n * 32, p);
        }
        __builtin_amdgcn_s_setprio(0);
        if (ahead) {
#pragma unroll
          for (int q = 0; q < QT; ++q) s[q] = s1[q];
          look(TAIL && kc + (n + 2) * 32 > all, kc + (n + 1) * 32);
        }
      }
      if (TAIL && odd_tile[buf] == kc)
        for (int n = 0; n < NS; ++n)
          w.add_specials(vp + (int64_t)(kc + n * 32) * a.v_ld, a.v_ld, sp.k_lim - kc - n * 32, a.dim, kc + n * 32);
      kc += KT;
    };
    while (kc + 4 * KT <= all && kc + 3 * KT < ke) {     // three at a time: LDS addresses are constants
      tile(std::false_type{}, 0, true);
      tile(std::false_type{}, 1, true);
      tile(std::false_type{}, 2, true);
    }
    for (int buf = 0; kc < ke; buf = buf == 2 ? 0 : buf + 1) tile(std::true_type{}, buf, kc + KT < ke);
  }
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    if (a.parts == 1) {
      w.store(q, static_cast<T*>(a.out) + qrow[q] * a.o_ld + head[q] * a.o_hd, a.dim, ok[q]);
    } else {
      const int64_t i = ((int64_t)part * a.s.q_rows + qrow[q]) * a.heads + head[q];
      w.store_part(q, a.part_o + i * a.dim, a.part_rl + i, a.dim, ok[q]);
    }
  }
}

// ---------------------------------------------------------------------------
// Few queries to a sequence (single tokens): a workgroup takes 32 rows, the
// queries of all heads of one key head, so that the keys are read once for
// the group; its NW waves take different tiles of 32 keys, each on its own (no
// barrier inside the loop), and join their O, m and l through LDS at the end.
// Memory bound: K goes straight to registers in operand layout (16 bytes of a
// row to a lane), V through a wave's own LDS tile for the transposed reads,
// the next tile's loads in flight meanwhile.  64 tokens over 500 .. 8000 keys,
// 32 heads on 8 of 128, 1.14 GB: 233 us, 4.9 TB/s.
template <typename T, int D, int NW>
__device__ __forceinline__ void few_body(const vrs_attention_args& a) {
  using E = Elt<T>;
  using G = typename E::group;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = 32 * CH / 64;                 // V chunks of a lane
  constexpr int OL = D + 4;                        // O row in LDS (float32)
  constexpr int V_BYTES = NW * 32 * D * (int)sizeof(T), O_BYTES = NW * 32 * OL * 4;
  __shared__ __attribute__((aligned(16))) char mem[V_BYTES > O_BYTES ? V_BYTES : O_BYTES];
  __shared__ float sR[NW][32], sl[NW][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // no two workgroups share keys: in the order of launch, round the XCDs, the
  // sequences with the most keys first
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv;
  const int part = rest % a.parts;
  const SeqSpan sp = ranked_seq(a.s, rest / a.parts);
  const int G_ = a.heads / a.kv;
  const int64_t rows = (int64_t)sp.q_len * G_;
  T* sV = reinterpret_cast<T*>(mem) + wave * 32 * D;
  float* sO = reinterpret_cast<float*>(mem);

  const Log2 u(a.c);
  // row tiles of the sequence, one workgroup each (and more than were counted on, in turn)
  for (int64_t r0 = blockIdx.y * 32; r0 < rows; r0 += gridDim.y * 32) {
    Wave<T, D, 1> w;
    w.init(u);
    const int64_t pr = min(r0 + w.l32, rows - 1);
    const bool ok = r0 + w.l32 < rows;
    const int j = (int)(pr / G_), h = hk * G_ + (int)(pr - (int64_t)j * G_);
    const int64_t row = sp.q0 + j;
    const int lim = visible(sp, j, a.causal);
    w.lim[0] = lim;
    w.load_q(0, static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd, a.dim, ok);
    const int lim_min = __builtin_amdgcn_readfirstlane(lim), lim_max = __builtin_amdgcn_readlane(lim, 31);
    int kb, ke;
    part_of(lim_max, part, a.parts, 32, kb, ke);

    const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
    const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
    G kr[D / 16];
    u32x4_t vr[IT];
    uint32_t ko[D / 16], vo[IT];           // offsets in a tile; elements past the head read 0
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = i * 16 + w.hh * 8;
      ko[i] = d < a.dim ? (uint32_t)(w.l32 * (int)a.k_ld + d) * (uint32_t)sizeof(T) : kOOB;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int it = lane + i * 64, r = it / CH, ch = it % CH;
      vo[i] = ch * PER < a.dim ? (uint32_t)(r * (int)a.v_ld + ch * PER) * (uint32_t)sizeof(T) : kOOB;
    }
    auto load = [&](int kc) {              // keys past the sequence's last are masked, whatever they read
      const int n = min(32, sp.k_lim - kc);
      const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
      const auto rv = make_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((n - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) kr[i] = E::bload(rk, ko[i], 0);
#pragma unroll
      for (int i = 0; i < IT; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, vo[i], 0, 0);
    };
    int kc = kb + wave * 32;
    if (kc < ke) load(kc);
    while (kc < ke) {
      f32x16_t s[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s[0] = mfma32_k16(kr[i], w.qf[0][i], s[0]);
      const int at = kc;
      const bool masked = at + 32 > lim_min;
      bool bad = false;
      if (masked) {
#pragma unroll
        for (int i = 0; i < IT; ++i) bad |= clean<T>(vr[i]);
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int it = lane + i * 64, r = it / CH, ch = it % CH;
        *reinterpret_cast<u32x4_t*>(sV + r * D + (ch ^ Lds<T, D>::vswz(r)) * PER) = vr[i];
      }
      __builtin_amdgcn_wave_barrier();     // the wave's own tile: order alone is needed
      kc += NW * 32;
      if (kc < ke) load(kc);
      if (masked) w.mask(0, s[0], at);
      const float t[1] = {w.top(s[0])};
      w.follow(t, u);
      const typename Wave<T, D, 1>::P p[1] = {w.probs(0, s[0], u)};
      w.pv(sV, 0, p);
      if (__any(bad)) w.add_specials(vp + (int64_t)at * a.v_ld, a.v_ld, sp.k_lim - at, a.dim, at);
      __builtin_amdgcn_wave_barrier();
    }
    // join the waves: the largest reference, sums and O scaled to it
    const float lt = sum32(w.l[0]);
    __syncthreads();                       // every wave is done with its V tile
    if (w.hh == 0) {
      sR[wave][w.l32] = w.R[0];
      sl[wave][w.l32] = lt;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t*>(&sO[(wave * 32 + w.l32) * OL + d * 32 + g * 8 + w.hh * 4]) =
            (f32x4_t){w.o[0][d][4 * g], w.o[0][d][4 * g + 1], w.o[0][d][4 * g + 2], w.o[0][d][4 * g + 3]};
    __syncthreads();
    // 2 NW threads to a row, 4 elements at a time
    const int rr = threadIdx.x / (2 * NW), e0 = threadIdx.x % (2 * NW) * 4;
    if (r0 + rr < rows) {
      const int jj = (int)((r0 + rr) / G_), ho = hk * G_ + (int)(r0 + rr - (int64_t)jj * G_);
      const int64_t orow = sp.q0 + jj;
      float mx = sR[0][rr];
#pragma unroll
      for (int i = 1; i < NW; ++i) mx = fmaxf(mx, sR[i][rr]);
      float f[NW], lsum = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {       // a wave without keys has l = 0, O = 0
        f[i] = u.factor(sR[i][rr], mx);
        lsum += f[i] * sl[i][rr];
      }
      const float inv = a.parts > 1 ? 1.f : share(lsum, visible(sp, jj, a.causal));
      const int64_t at = ((int64_t)part * a.s.q_rows + orow) * a.heads + ho;
      if (a.parts > 1 && e0 == 0) a.part_rl[at] = make_float2(mx, lsum);
      T* out = static_cast<T*>(a.out) + orow * a.o_ld + ho * a.o_hd;
      for (int e = e0; e < a.dim; e += 8 * NW) {
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) v += f[i] * *reinterpret_cast<const f32x4_t*>(&sO[(i * 32 + rr) * OL + e]);
        v *= inv;
        if (a.parts > 1) {
          *reinterpret_cast<f32x4_t*>(a.part_o + at * a.dim + e) = v;
        } else if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<f32x4_t*>(out + e) = v;
        } else {
          *reinterpret_cast<u32x2_t*>(out + e) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        }
      }
    }
    __syncthreads();                       // sO is the V tiles of the next rows
  }
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
    prompt_body<T, D, KT, QT, NW>(a);                                                                                         \
  }
#define VRS_ATTENTION_FEW(TN, T, D, NW, WPS)                                                                               \
  extern "C" __global__ __launch_bounds__(64 * NW, WPS) void vrs_attention_few_##TN##_d##D##_w##NW(vrs_attention_args a) { \
    few_body<T, D, NW>(a);                                                                                                 \
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
