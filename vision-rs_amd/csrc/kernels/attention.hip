// Attention over packed sequences and over a cache, for gfx950:
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys j < lim_i of the query's sequence (causal: those at or before
// its own place; else all), with grouped heads (heads / kv_heads queries to a
// key head) and head sizes up to 64 or 128 (shorter ones padded by loads that
// read zeros).
//
// Both kernels work in wave tiles of 32 queries x 32 keys:
//   S^T(keys x queries) = K Q^T     on 32x32 MFMA, K rows as A, Q^T as B
//   p = exp2(s c - m c)             c = scale log2 e; one FMA and one v_exp
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

template <typename T, int D>
struct Wave {
  using E = Elt<T>;
  using G = typename E::group;
  static constexpr int PER = 16 / (int)sizeof(T);   // elements of a chunk
  G qf[D / 16];
  f32x16_t o[D / 32];
  float m, l;          // running maximum (raw scores) and this lane's share of the sum
  int l32, hh;

  __device__ __forceinline__ void init() {
    l32 = threadIdx.x & 31;
    hh = (threadIdx.x >> 5) & 1;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
  }
  // Q^T operand: 8 elements at s * 16 + hh * 8 of the lane's query
  __device__ __forceinline__ void load_q(const T* q, int dim, bool ok) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const int d = s * 16 + hh * 8;
      qf[s] = ok && d < dim ? E::load(q + d) : E::zero();
    }
  }
  // register r of an S^T accumulator: key of the 32
  __device__ __forceinline__ int key_of(int r) const { return (r >> 2) * 8 + hh * 4 + (r & 3); }

  // running maximum and sum over NS * 32 keys starting at kc, those from lim on masked; s becomes p
  template <int NS>
  __device__ __forceinline__ void softmax(f32x16_t (&s)[NS], int kc, int lim, bool masked, float c) {
    if (masked) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] = kc + n * 32 + key_of(r) < lim ? s[n][r] : -INFINITY;
    }
    float t = -INFINITY;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) t = fmaxf(t, s[n][r]);
    t = max32(t);
    if (__any((t - m) * c > kTau)) {
      // (a first maximum: t - -inf; lanes without any key yet keep -inf and factor 1)
      const float mn = fmaxf(m, t);
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) o[d] *= alpha;
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][r], c, -mc));
        if constexpr (sizeof(T) == 4) l += s[n][r];
      }
  }

  // S^T of the 32 keys from `row` of a K tile in LDS
  __device__ __forceinline__ f32x16_t scores(const T* sK, int row) const {
    f32x16_t s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
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
      s = mfma32_k16(kf, qf[i], s);
    }
    return s;
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
  // Adds what the infinities and NaN among 32 keys (rows of v, n of them, dim elements) give the
  // queries that see them (bit r of seen: key_of(r)): for each sign, indicators of such values times
  // indicators of seen keys.  A NaN counts as an infinity of either sign (inf - inf).  Reads memory
  // again: rare, so small code rather than fast.
  __device__ __forceinline__ void add_specials(const T* v, int64_t ld, int n, int dim, uint32_t seen) {
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
          const int key = (r >> 2) * 8 + hh * 4 + (r & 3), e = d * 32 + l32;
          const float x = key < n && e < dim ? E::to_f(v[key * ld + e]) : 0.f;
          count = __builtin_amdgcn_mfma_f32_32x32x2f32(x != x || x == inf ? 1.f : 0.f, (seen >> r) & 1 ? 1.f : 0.f, count, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] += count[r] > 0.f ? inf : 0.f;
      }
    }
  }
  // registers of the 32 keys from kc that lie before lim
  __device__ __forceinline__ uint32_t seen_mask(int kc, int lim) const {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) m |= kc + key_of(r) < lim ? 1u << r : 0u;
    return m;
  }

  // O^T += V^T P^T over the 32 keys from `row` of a V tile, p their probabilities
  __device__ __forceinline__ void pv(const T* sV, int row, const f32x16_t& p) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        G pf;
        pf.v = (u32x4_t){pack_bf16x2(p[8 * ks], p[8 * ks + 1]), pack_bf16x2(p[8 * ks + 2], p[8 * ks + 3]),
                         pack_bf16x2(p[8 * ks + 4], p[8 * ks + 5]), pack_bf16x2(p[8 * ks + 6], p[8 * ks + 7])};
#pragma unroll
        for (int j = 0; j < 4; ++j)    // sum of the rounded pairs
          l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v_t, (uint32_t)pf.v[j]),
                                              __builtin_bit_cast(bf16x2v_t, 0x3f803f80u), l, false);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const G vf = vt(sV, row + ks * 16, d);
          o[d] = mfma32_k16(vf, pf, o[d]);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v1(sV, row, r, d), p[r], o[d], 0, 0, 0);
    }
  }

  // O / l of the lane's query to `out` (element type), `dim` elements; no key seen: zeros
  __device__ __forceinline__ void store(T* out, int dim, bool ok) {
    const float lt = sum32(l);
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int e = d * 32 + g * 8 + hh * 4;
          const f32x4_t v = {o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv};
          if (ok && e < dim) *reinterpret_cast<f32x4_t*>(out + e) = v;
        }
      } else {
        // two quads of 4: the halves swapped so that each lane has 8 elements in a row
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          u32x2_t a = {pack_bf16x2(o[d][4 * g] * inv, o[d][4 * g + 1] * inv),
                       pack_bf16x2(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv)};
          u32x2_t b = {pack_bf16x2(o[d][4 * g + 4] * inv, o[d][4 * g + 5] * inv),
                       pack_bf16x2(o[d][4 * g + 6] * inv, o[d][4 * g + 7] * inv)};
          const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
          const auto y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
          const int e = d * 32 + g * 8 + hh * 8;
          if (ok && e < dim) *reinterpret_cast<u32x4_t*>(out + e) = (u32x4_t){x[0], y[0], x[1], y[1]};
        }
      }
    }
  }

  // the unfinished query to a workspace: O (float32), running maximum in log2 units, sum
  __device__ __forceinline__ void store_part(float* po, float2* pml, int dim, float c, bool ok) {
    const float lt = sum32(l);
    if (ok && hh == 0) *pml = make_float2(m == -INFINITY ? -INFINITY : m * c, lt);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = d * 32 + g * 8 + hh * 4;
        const f32x4_t v = {o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
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

// ---------------------------------------------------------------------------
// Prompts: a workgroup of 4 waves takes 128 queries of one head, a wave 32;
// K and V tiles are shared through LDS, double buffered, the next tile's loads
// in flight in registers while this one is computed.
template <typename T, int D, int KT>
__device__ __forceinline__ void prompt_body(const vrs_attention_args& a) {
  constexpr int NT = 256, BM = 128;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = KT * CH / NT;                 // chunks a thread stages of K, and of V
  __shared__ __attribute__((aligned(16))) T smem[2][2][KT * D];
  __shared__ int odd_tile[2];     // first key of the tile that a buffer holds, if it had values not finite
  const int tid = threadIdx.x, wave = tid >> 6;
  // heads outermost: an XCD's workgroups read few heads' keys; a head's late
  // query tiles (the longest, when causal) first
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int part = logical % a.parts;
  const int rest = logical / a.parts;
  const int tile_id = a.tiles - 1 - rest % a.tiles, h = rest / a.tiles;
  // sequence i's query tiles are ids floor(q_start[i] / BM) + i + 0, 1, ...: enough
  // ids for each whatever the lengths, so no table of tiles is needed
  auto first = [&](int i) { return min(max(a.s.q_start[i], 0), a.s.q_rows) / BM + i; };
  if (tile_id < first(0)) return;
  const int sq = find_seq(a.s.n, tile_id, first);
  const SeqSpan sp = seq_span(a.s, sq);
  const int j0 = (tile_id - first(sq)) * BM;
  if (j0 < 0 || j0 >= sp.q_len) return;
  const int hk = h / (a.heads / a.kv);

  Wave<T, D> w;
  w.init();
  const int j = j0 + wave * 32 + w.l32;
  const bool ok = j < sp.q_len;
  const int lim = visible(sp, min(j, sp.q_len - 1), a.causal);
  w.load_q(static_cast<const T*>(a.q) + (int64_t)(sp.q0 + j) * a.q_ld + h * a.q_hd, a.dim, ok);

  int kb, ke;
  part_of(visible(sp, min(j0 + BM, sp.q_len) - 1, a.causal), part, a.parts, KT, kb, ke);
  const int lim_min = __builtin_amdgcn_readfirstlane(lim), lim_max = __builtin_amdgcn_readlane(lim, 31);

  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
  u32x4_t kr[IT], vr[IT];
  // keys past the sequence's last and elements past the head read 0
  auto load = [&](int kc) {
    const int rows = min(KT, sp.k_lim - kc);
    const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((rows - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
    const auto rv = make_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((rows - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int it = tid + i * NT, row = it / CH, ch = it % CH;
      const bool in = ch * PER < a.dim && row < rows;
      kr[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, in ? (uint32_t)(row * (int)a.k_ld + ch * PER) * sizeof(T) : kOOB, 0, 0);
      vr[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, in ? (uint32_t)(row * (int)a.v_ld + ch * PER) * sizeof(T) : kOOB, 0, 0);
    }
  };
  // keys that every query of the workgroup sees
  const int all = visible(sp, j0, a.causal);
  auto stage = [&](int buf, int kc) {
    if (kc + KT > all) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < IT; ++i) bad |= clean<T>(vr[i]);
      if (bad) odd_tile[buf] = kc;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int it = tid + i * NT, row = it / CH, ch = it % CH;
      *reinterpret_cast<u32x4_t*>(&smem[buf][0][row * D + (ch ^ Lds<T, D>::kswz(row)) * PER]) = kr[i];
      *reinterpret_cast<u32x4_t*>(&smem[buf][1][row * D + (ch ^ Lds<T, D>::vswz(row)) * PER]) = vr[i];
    }
  };
  if (kb < ke) {
    load(kb);
    if (tid < 2) odd_tile[tid] = -1;
    __syncthreads();
    stage(0, kb);
    __syncthreads();
    int buf = 0;
    for (int kc = kb; kc < ke; kc += KT, buf ^= 1) {
      const bool more = kc + KT < ke;
      if (more) load(kc + KT);
      if (kc < lim_max) {
        const T* sK = smem[buf][0];
        const T* sV = smem[buf][1];
        f32x16_t s[KT / 32];
#pragma unroll
        for (int n = 0; n < KT / 32; ++n) s[n] = w.scores(sK, n * 32);
        w.softmax(s, kc, lim, kc + KT > lim_min, a.c);
#pragma unroll
        for (int n = 0; n < KT / 32; ++n) w.pv(sV, n * 32, s[n]);
        if (odd_tile[buf] == kc)
          for (int n = 0; n < KT; n += 32)
            w.add_specials(vp + (int64_t)(kc + n) * a.v_ld, a.v_ld, sp.k_lim - kc - n, a.dim, w.seen_mask(kc + n, lim));
      }
      if (more) stage(buf ^ 1, kc + KT);
      __syncthreads();
    }
  }
  const int64_t row = sp.q0 + j;
  if (a.parts == 1) {
    w.store(static_cast<T*>(a.out) + row * a.o_ld + h * a.o_hd, a.dim, ok);
  } else {
    const int64_t at = ((int64_t)part * a.s.q_rows + row) * a.heads + h;
    w.store_part(a.part_o + at * a.dim, a.part_ml + at, a.dim, a.c, ok);
  }
}

// ---------------------------------------------------------------------------
// Few queries to a sequence (single tokens): a workgroup takes 32 rows, the
// queries of all heads of one key head, so that the keys are read once for
// the group; its 4 waves take different tiles of 32 keys, each on its own (no
// barrier inside the loop), and join their O, m and l through LDS at the end.
// Memory bound: K goes straight to registers in operand layout (16 bytes of a
// row to a lane), V through a wave's own LDS tile for the transposed reads,
// the next tile's loads in flight meanwhile.
template <typename T, int D>
__device__ __forceinline__ void few_body(const vrs_attention_args& a) {
  using E = Elt<T>;
  using G = typename E::group;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = 32 * CH / 64;                 // V chunks of a lane
  constexpr int OL = D + 4;                        // O row in LDS (float32)
  constexpr int V_BYTES = 4 * 32 * D * (int)sizeof(T), O_BYTES = 4 * 32 * OL * 4;
  __shared__ __attribute__((aligned(16))) char mem[V_BYTES > O_BYTES ? V_BYTES : O_BYTES];
  __shared__ float sm[4][32], sl[4][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int logical = xcd_remap(blockIdx.x, gridDim.x);
  const int part = logical % a.parts;
  const int rest = logical / a.parts;
  const int hk = rest % a.kv, sq = rest / a.kv;
  const SeqSpan sp = seq_span(a.s, sq);
  const int G_ = a.heads / a.kv;
  const int64_t rows = (int64_t)sp.q_len * G_;
  T* sV = reinterpret_cast<T*>(mem) + wave * 32 * D;
  float* sO = reinterpret_cast<float*>(mem);

  // row tiles of the sequence, one workgroup each (and more than were counted on, in turn)
  for (int64_t r0 = blockIdx.y * 32; r0 < rows; r0 += gridDim.y * 32) {
    Wave<T, D> w;
    w.init();
    const int64_t pr = min(r0 + w.l32, rows - 1);
    const bool ok = r0 + w.l32 < rows;
    const int j = (int)(pr / G_), h = hk * G_ + (int)(pr - (int64_t)j * G_);
    const int64_t row = sp.q0 + j;
    const int lim = visible(sp, j, a.causal);
    w.load_q(static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd, a.dim, ok);
    const int lim_min = __builtin_amdgcn_readfirstlane(lim), lim_max = __builtin_amdgcn_readlane(lim, 31);
    int kb, ke;
    part_of(lim_max, part, a.parts, 32, kb, ke);

    const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
    const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
    G kr[D / 16];
    u32x4_t vr[IT];
    auto load = [&](int kc) {
      const int n = min(32, sp.k_lim - kc);
      const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
      const auto rv = make_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((n - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int d = i * 16 + w.hh * 8;
        kr[i] = E::bload(rk, d < a.dim && w.l32 < n ? (uint32_t)(w.l32 * (int)a.k_ld + d) * sizeof(T) : kOOB, 0);
      }
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int it = lane + i * 64, r = it / CH, ch = it % CH;
        vr[i] = __builtin_amdgcn_raw_buffer_load_b128(
            rv, ch * PER < a.dim && r < n ? (uint32_t)(r * (int)a.v_ld + ch * PER) * sizeof(T) : kOOB, 0, 0);
      }
    };
    int kc = kb + wave * 32;
    if (kc < ke) load(kc);
    while (kc < ke) {
      f32x16_t s[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s[0] = mfma32_k16(kr[i], w.qf[i], s[0]);
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
      kc += 128;
      if (kc < ke) load(kc);
      w.softmax(s, at, lim, masked, a.c);
      w.pv(sV, 0, s[0]);
      if (__any(bad)) w.add_specials(vp + (int64_t)at * a.v_ld, a.v_ld, sp.k_lim - at, a.dim, w.seen_mask(at, lim));
      __builtin_amdgcn_wave_barrier();
    }
    // join the four waves: the largest maximum, sums and O scaled to it
    const float lt = sum32(w.l);
    __syncthreads();                       // every wave is done with its V tile
    if (w.hh == 0) {
      sm[wave][w.l32] = w.m;
      sl[wave][w.l32] = lt;
    }
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4_t*>(&sO[(wave * 32 + w.l32) * OL + d * 32 + g * 8 + w.hh * 4]) =
            (f32x4_t){w.o[d][4 * g], w.o[d][4 * g + 1], w.o[d][4 * g + 2], w.o[d][4 * g + 3]};
    __syncthreads();
    // 8 threads to a row, 4 elements at a time
    const int rr = threadIdx.x >> 3, e0 = (threadIdx.x & 7) * 4;
    if (r0 + rr < rows) {
      const int jj = (int)((r0 + rr) / G_), ho = hk * G_ + (int)(r0 + rr - (int64_t)jj * G_);
      const int64_t orow = sp.q0 + jj;
      const float mx = fmaxf(fmaxf(sm[0][rr], sm[1][rr]), fmaxf(sm[2][rr], sm[3][rr]));
      float f[4], lsum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {        // a wave without keys has l = 0, O = 0
        f[i] = sm[i][rr] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sm[i][rr] - mx) * a.c);
        lsum += f[i] * sl[i][rr];
      }
      const float inv = a.parts > 1 ? 1.f : lsum == 0.f ? 0.f : 1.f / lsum;
      const int64_t at = ((int64_t)part * a.s.q_rows + orow) * a.heads + ho;
      if (a.parts > 1 && (threadIdx.x & 7) == 0) a.part_ml[at] = make_float2(mx == -INFINITY ? mx : mx * a.c, lsum);
      T* out = static_cast<T*>(a.out) + orow * a.o_ld + ho * a.o_hd;
      for (int e = e0; e < a.dim; e += 32) {
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) v += f[i] * *reinterpret_cast<const f32x4_t*>(&sO[(i * 32 + rr) * OL + e]);
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
// Joins the parts of the keys: a wave takes one (row, head).
template <typename T>
__device__ __forceinline__ void join_body(const vrs_attention_args& a) {
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = id / a.heads;
  const int h = (int)(id - row * a.heads);
  if (row >= a.s.q_rows || row < a.s.q_start[0]) return;
  const int sq = find_seq(a.s.n, (int)row, [&](int i) { return a.s.q_start[i]; });
  const SeqSpan sp = seq_span(a.s, sq);
  if (row < sp.q0 || row >= sp.q0 + sp.q_len) return;
  const int64_t step = (int64_t)a.s.q_rows * a.heads;
  float mx = -INFINITY;
  for (int p = 0; p < a.parts; ++p) mx = fmaxf(mx, a.part_ml[p * step + id].x);
  float l = 0.f;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  const int e = lane * 4;
  for (int p = 0; p < a.parts; ++p) {
    const float2 ml = a.part_ml[p * step + id];
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
    l += f * ml.y;
    if (e < a.dim) v += f * *reinterpret_cast<const f32x4_t*>(a.part_o + (p * step + id) * a.dim + e);
  }
  v *= l == 0.f ? 0.f : 1.f / l;
  if (e >= a.dim) return;
  T* out = static_cast<T*>(a.out) + row * a.o_ld + h * a.o_hd + e;
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4_t*>(out) = v;
  else *reinterpret_cast<u32x2_t*>(out) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
}  // namespace

#define VRS_ATTENTION(TN, T, D, KT)                                                                          \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_attention_prompt_##TN##_d##D(vrs_attention_args a) { \
    prompt_body<T, D, KT>(a);                                                                                \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void vrs_attention_few_##TN##_d##D(vrs_attention_args a) { \
    few_body<T, D>(a);                                                                                       \
  }
VRS_ATTENTION(bf16, bf16_t, 64, 64)
VRS_ATTENTION(bf16, bf16_t, 128, 64)
VRS_ATTENTION(f32, float, 64, 32)
VRS_ATTENTION(f32, float, 128, 32)
extern "C" __global__ __launch_bounds__(256) void vrs_attention_join_bf16(vrs_attention_args a) { join_body<bf16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_attention_join_f32(vrs_attention_args a) { join_body<float>(a); }
