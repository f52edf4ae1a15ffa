// Attention that keys receive, for gfx950:
//   acc_j = decay acc_j + sum_i p_ij,  p_ij = softmax_j(scale q_i . k_j)
// over the queries of a sequence and the heads of a key head.  A weight needs its
// row's whole sum before it counts, so there are two steps: the rows' references
// and sums (softmax statistics, see Log2), then the sum over the rows of each key.
//
// Few rows to a key head (single tokens): the first step leaves the scores, which
// are a small part of the keys' bytes, and the second reads those.  Many: the
// second multiplies again, a wave holding 32 keys while the queries pass by.
#include "attention_wave.h"

namespace {

// Stage 1, few rows: a workgroup of 4 waves takes 32 rows of one key head against a
// part of the keys, its waves every fourth 32 of them.  Memory bound: K is loaded by
// whole rows (a lane's operand straight from memory touches a row in eight
// instructions, and the lines are gone from L1 in between: 165 us instead of 128
// for the scores of 64 tokens over 500 .. 8000 keys, 32 heads on 8 of 128) and turned in a wave's own
// LDS tile, the next tile's loads in flight meanwhile.
template <typename T, int D>
__device__ __forceinline__ void scores_body(const vrs_weights_args& a) {
  constexpr int NW = 4, CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T), IT = 32 * CH / 64;
  __shared__ __attribute__((aligned(16))) T tiles[NW][32 * D];
  __shared__ float sR[NW][32], sl[NW][32];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  T* const sK = tiles[wave];
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv, part = rest % a.parts;
  const SeqSpan sp = ranked_seq(Sequences{a.s}, rest / a.parts);
  const int G_ = a.heads / a.kv;
  const int64_t rows = (int64_t)sp.q_len * G_;
  const Log2 u(a.c);
  for (int64_t r0 = (int64_t)blockIdx.y * 32; r0 < rows; r0 += (int64_t)gridDim.y * 32) {
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
    u32x4_t held[IT];
    uint32_t ko[IT];                       // offsets in a tile; elements past the head read 0
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int it = lane + i * 64, r = it / CH, ch = it % CH;
      ko[i] = ch * PER < a.dim ? (uint32_t)(r * (int)a.k_ld + ch * PER) * (uint32_t)sizeof(T) : kOOB;
    }
    auto load = [&](int kc) {              // keys past the sequence's last are masked, whatever they read
      const int n = min(32, sp.k_lim - kc);
      const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
      for (int i = 0; i < IT; ++i) held[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, ko[i], 0, 0);
    };
    float* keep = a.scores + (row * a.heads + h) * a.s_ld;
    int kc = kb + wave * 32;
    if (kc < ke) load(kc);
    while (kc < ke) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int it = lane + i * 64, r = it / CH, ch = it % CH;
        *reinterpret_cast<u32x4_t*>(sK + r * D + (ch ^ Lds<T, D>::kswz(r)) * PER) = held[i];
      }
      __builtin_amdgcn_wave_barrier();     // the wave's own tile: order alone is needed
      const int at = kc;
      kc += NW * 32;
      if (kc < ke) load(kc);
      f32x16_t sc[1];
      w.scores(sK, 0, sc);
      __builtin_amdgcn_wave_barrier();
      f32x16_t& s = sc[0];
      if (at + 32 > lim_min) w.mask(0, s, at);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t key = at + g * 8 + w.hh * 4;
        const f32x4_t v = {s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
        if (ok && key < a.s_ld) *reinterpret_cast<f32x4_t*>(keep + key) = v;
      }
      const float t[1] = {w.top(s)};
      w.follow(t, u);
#pragma unroll
      for (int r = 0; r < 16; ++r) w.l[0] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], w.unit[0], -w.R[0]));
    }
    const float lt = sum32(w.l[0]);
    __syncthreads();                       // the last rows' statistics are read
    if (w.hh == 0) {
      sR[wave][w.l32] = w.R[0];
      sl[wave][w.l32] = lt;
    }
    __syncthreads();
    if (threadIdx.x < 32 && ok) {
      float mx = sR[0][w.l32], l = 0.f;
#pragma unroll
      for (int i = 1; i < NW; ++i) mx = fmaxf(mx, sR[i][w.l32]);
#pragma unroll
      for (int i = 0; i < NW; ++i) l += u.factor(sR[i][w.l32], mx) * sl[i][w.l32];
      a.rl[((int64_t)part * a.s.q_rows + row) * a.heads + h] = make_float2(mx, l);
    }
  }
}

// Streaming tiles of 64 rows (keys for the statistics, queries for the sums) in
// LDS, twice: a thread holds the next tile's chunks in registers while this one is
// in use, so that one barrier a tile is enough.
template <typename T, int D>
struct Stream {
  using G = typename Elt<T>::group;
  static constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T), IT = 64 * CH / 256, TILE = 64 * D;
  u32x4_t held[IT];
  __device__ __forceinline__ static int row(int i) { return (i * 256 + (int)threadIdx.x) / CH; }
  __device__ __forceinline__ static int elt(int i) { return (i * 256 + (int)threadIdx.x) % CH * PER; }
  __device__ __forceinline__ void put(T* tile) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = row(i);
      *reinterpret_cast<u32x4_t*>(tile + r * D + (((i * 256 + (int)threadIdx.x) % CH) ^ Lds<T, D>::kswz(r)) * PER) = held[i];
    }
  }
};

// Stage 1, many rows: a workgroup of 4 waves takes 128 rows, which the keys pass by.
// 4096 causal queries, 32 heads on 8 of 128: 89 us, 712 cycles a tile of 32 x 32 on a
// SIMD: 256 of matrix instructions and 430 of vector ones (16 v_exp at four times an
// instruction's cycles, as many FMAs and additions, the maximum), which the waves of
// a SIMD hardly overlap.  Keys straight from memory to each wave's registers: 265 us.
template <typename T, int D>
__device__ __forceinline__ void stats_body(const vrs_weights_args& a) {
  using S = Stream<T, D>;
  __shared__ __attribute__((aligned(16))) T tile[2][S::TILE];
  const int wave = threadIdx.x >> 6;
  const int hk = blockIdx.x % a.kv, rest = blockIdx.x / a.kv, part = rest % a.parts;
  const int group = a.heads / a.kv;
  const TilePlace at = place_tile<128>(Sequences{a.s}, group, rest / a.parts);
  if (at.tile < 0) return;
  const SeqSpan sp = at.sp;
  const int64_t rows = (int64_t)sp.q_len * group;
  const int tiles = (int)((rows + 127) / 128);
  if (at.tile >= tiles) return;
  const int64_t r0 = (int64_t)(tiles - 1 - at.tile) * 128;       // late rows (causal: the most keys) first
  const Log2 u(a.c);
  Wave<T, D, 1> w;
  w.init(u);
  const int64_t r = r0 + wave * 32 + w.l32, pr = min(r, rows - 1);
  const bool ok = r < rows;
  const int j = (int)(pr / group), h = hk * group + (int)(pr - (int64_t)j * group);
  const int64_t row = sp.q0 + j;
  w.lim[0] = visible(sp, j, a.causal);
  w.load_q(0, static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd, a.dim, ok);
  int kb, ke;
  part_of(visible(sp, (int)((min(r0 + 128, rows) - 1) / group), a.causal), part, a.parts, 64, kb, ke);
  const int all = __builtin_amdgcn_readlane(w.lim[0], 0), mine = __builtin_amdgcn_readlane(w.lim[0], 31);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  S st;
  auto load = [&](int kc) {              // keys past the sequence's last read 0 and are masked
    const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((min(64, sp.k_lim - kc) - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
    for (int i = 0; i < S::IT; ++i)
      st.held[i] = __builtin_amdgcn_raw_buffer_load_b128(
          rk, S::elt(i) < a.dim ? (uint32_t)(S::row(i) * (int)a.k_ld + S::elt(i)) * (uint32_t)sizeof(T) : kOOB, 0, 0);
  };
  if (kb < ke) {
    load(kb);
    st.put(tile[0]);
    if (kb + 64 < ke) load(kb + 64);
    __syncthreads();
    for (int kc = kb, buf = 0; kc < ke; kc += 64, buf ^= 1) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int at0 = kc + n * 32;
        if (at0 >= mine) break;
        f32x16_t s[1];
        w.scores(tile[buf], n * 32, s);
        if (at0 + 32 > all) w.mask(0, s[0], at0);
        const float t[1] = {w.top(s[0])};
        w.follow(t, u);
#pragma unroll
        for (int i = 0; i < 16; ++i) w.l[0] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], w.unit[0], -w.R[0]));
      }
      if (kc + 64 < ke) st.put(tile[buf ^ 1]);
      if (kc + 128 < ke) load(kc + 128);
      __syncthreads();
    }
  }
  const float lt = sum32(w.l[0]);
  if (w.hh == 0 && ok) a.rl[((int64_t)part * a.s.q_rows + row) * a.heads + h] = make_float2(w.R[0], lt);
}

// A row's reference and sum over the parts of its keys.
__device__ __forceinline__ float2 joined(const vrs_weights_args& a, const Log2& u, int64_t id) {
  const int64_t step = (int64_t)a.s.q_rows * a.heads;
  float mx = kNone, l = 0.f;
#pragma unroll 8
  for (int p = 0; p < a.parts; ++p) mx = fmaxf(mx, a.rl[p * step + id].x);
#pragma unroll 8
  for (int p = 0; p < a.parts; ++p) {
    const float2 rl = a.rl[p * step + id];
    l += u.factor(rl.x, mx) * rl.y;
  }
  return make_float2(mx, l);
}

// Between the stages, many rows whose keys are in parts: a thread joins a row's parts and leaves them as the first.
// In stage 2 each tile of keys would do so again, with registers that its products need: 100 queries over 4000 keys,
// 32 heads on 8 of 128, 16 parts: 60 us a call, 35 with this launch; a prompt of 4096, whose rows have one part: 14
// registers of stage 2 spilled and 112 us, 2 and 100.
__device__ __forceinline__ void rows_body(const vrs_weights_args& a) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)a.s.q_rows * a.heads) return;
  a.rl[id] = joined(a, Log2(a.c), id);
}

// Stage 2 from the scores: a thread takes 4 keys, 256 apart, and passes over the rows.
// 64 tokens over 500 .. 8000 keys: 20 us (one key a thread: 37).
template <typename T>
__device__ __forceinline__ void sum_body(const vrs_weights_args& a) {
  constexpr int RB = 32, KT = 4;
  __shared__ f32x4_t stat[RB];                // reference, 1 / sum, unit, keys seen (as bits)
  const int hk = blockIdx.x % a.kv;
  const SeqSpan sp = seq_span(a.s, blockIdx.x / a.kv);
  const int G_ = a.heads / a.kv;
  const int rows = (int)min((int64_t)sp.q_len * G_, (int64_t)0x7fffffff);
  const Log2 u(a.c);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  float* acc = a.acc + sp.k0 * a.acc_ld + hk * a.acc_hd;
  for (int64_t k0 = (int64_t)blockIdx.y * 256 * KT; k0 < sp.k_lim; k0 += (int64_t)gridDim.y * 256 * KT) {
    const int64_t key = k0 + threadIdx.x;
    float sum[KT], old[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      sum[t] = 0.f;
      old[t] = a.decay != 0.f && key + t * 256 < sp.k_lim ? acc[(key + t * 256) * a.acc_ld] : 0.f;
    }
    for (int r0 = 0; r0 < rows; r0 += RB) {
      __syncthreads();
      const int r = r0 + threadIdx.x;
      if (threadIdx.x < RB && r < rows) {
        const int j = r / G_;
        const int lim = visible(sp, j, a.causal);
        const float2 rl = joined(a, u, ((int64_t)sp.q0 + j) * a.heads + hk * G_ + (r - j * G_));
        stat[threadIdx.x] = (f32x4_t){rl.x, share(rl.y, lim), u.unit(rl.x), __int_as_float(lim)};
      }
      __syncthreads();
      const int n = min(RB, rows - r0);
      if (k0 + 256 * KT <= a.s_ld) {
        for (int i = 0; i < n; ++i) {
          const int j = (r0 + i) / G_, h = hk * G_ + (r0 + i - j * G_);
          const float* s = a.scores + (((int64_t)sp.q0 + j) * a.heads + h) * a.s_ld + key;
          const f32x4_t c = stat[i];
          float x[KT];
#pragma unroll
          for (int t = 0; t < KT; ++t) x[t] = s[t * 256];
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t], c[2], -c[0])) * c[1];
            sum[t] += key + t * 256 < __float_as_int(c[3]) ? p : 0.f;
          }
        }
      } else {      // more keys than were counted on: a key tile has all its scores or none (s_ld is whole tiles)
        for (int i = 0; i < n; ++i) {
          const int j = (r0 + i) / G_, h = hk * G_ + (r0 + i - j * G_);
          const int64_t row = (int64_t)sp.q0 + j;
          const f32x4_t c = stat[i];
          for (int t = 0; t < KT; ++t) {
            const int64_t at = key + t * 256;
            if (at >= __float_as_int(c[3])) break;
            const T* q = static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd;
            const T* k = kp + at * a.k_ld;
            float x = 0.f;
            for (int d = 0; d < a.dim; ++d) x = __builtin_fmaf(Elt<T>::to_f(q[d]), Elt<T>::to_f(k[d]), x);
            sum[t] += __builtin_amdgcn_exp2f(__builtin_fmaf(x, c[2], -c[0])) * c[1];
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < KT; ++t)
      if (key + t * 256 < sp.k_lim) acc[(key + t * 256) * a.acc_ld] = a.decay * old[t] + sum[t];
  }
}

// Stage 2 with the products again: a workgroup of 4 waves holds 128 keys, and a part
// of the rows that see them passes by in tiles of 64.  The same prompt: 100 .. 113 us
// (cards and their clocks differ).  Rows straight from memory to each wave: 919 us;
// their offsets by 64-bit arithmetic on vector registers, which makes the loads'
// buffer descriptors vectors too and puts a loop around each load: 130.  Three waves
// to a SIMD (168 registers, 2 more spilled): two 125, four 178 (37 spilled).
template <typename T, int D>
__device__ __forceinline__ void keys_body(const vrs_weights_args& a) {
  using E = Elt<T>;
  using G = typename E::group;
  using S = Stream<T, D>;
  __shared__ __attribute__((aligned(16))) T tile[2][S::TILE];
  __shared__ f32x4_t stat[2][64];             // reference, 1 / sum, unit, keys seen (as bits) of the tile's rows
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1;
  const int hk = blockIdx.x % a.kv, pair = blockIdx.x % (a.s.n * a.kv), part = blockIdx.x / (a.s.n * a.kv);
  const SeqSpan sp = seq_span(a.s, pair / a.kv);
  const int group = a.heads / a.kv;
  const float inv_group = 1.f / (float)group;
  const int64_t rows = (int64_t)sp.q_len * group;
  const Log2 u(a.c);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  float* acc = a.acc + sp.k0 * a.acc_ld + hk * a.acc_hd;
  for (int64_t k0 = (int64_t)blockIdx.y * 128; k0 < sp.k_lim; k0 += (int64_t)gridDim.y * 128) {
    // key tiles past those counted on have no place in the workspace: one workgroup takes all their rows
    const bool counted = k0 < (int64_t)a.s_ld;
    const int parts = counted ? a.key_parts : 1;
    if (part >= parts) return;
    const int kc = (int)k0 + wave * 32, n = min(32, max(sp.k_lim - kc, 1));
    G kr[D / 16];
    const auto rk = make_rsrc(kp + (int64_t)min(kc, sp.k_lim - 1) * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = i * 16 + hh * 8;
      kr[i] = E::bload(rk, d < a.dim ? (uint32_t)(l32 * (int)a.k_ld + d) * (uint32_t)sizeof(T) : kOOB, 0);
    }
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    // tiles from the first that has a row which sees key k0 on, shared out among the parts
    const int64_t skip = a.causal ? max((int64_t)0, k0 - ((int64_t)sp.k_len - sp.q_len)) * group : 0;
    // (divisions of 64 bits run on vector registers: what they give is made scalar again)
    const int t0 = __builtin_amdgcn_readfirstlane((int)(min(skip, rows) / 64)), t1 = (int)((rows + 63) >> 6);
    const int tb = __builtin_amdgcn_readfirstlane(t0 + (int)((int64_t)(t1 - t0) * part / parts));
    const int te = __builtin_amdgcn_readfirstlane(t0 + (int)((int64_t)(t1 - t0) * (part + 1) / parts));
    S st;
    // The next tile to load: its first query and that one's first head, and where a thread's chunks and its row of
    // the statistics lie from there.  Where 64 rows are whole queries these stay and the first query alone moves.
    int at = tb;
    int j0 = __builtin_amdgcn_readfirstlane((int)((int64_t)tb * 64 / group)), rem = (int)((int64_t)tb * 64 - (int64_t)j0 * group), sj, sh;
    uint32_t off[S::IT];
    auto places = [&]() {
#pragma unroll
      for (int i = 0; i < S::IT; ++i) {
        int h;
        const int j = fdivmod(rem + S::row(i), group, inv_group, h);
        off[i] = S::elt(i) < a.dim ? (uint32_t)(j * (int)a.q_ld + h * (int)a.q_hd + S::elt(i)) * (uint32_t)sizeof(T) : kOOB;
      }
      sj = fdivmod(rem + (int)(threadIdx.x & 63), group, inv_group, sh);
    };
    places();
    const int step = 64 / group, left = 64 % group;
    float2 rl;                                // a row's statistics, as they are stored
    int lim;
    auto load = [&]() {
      const auto rq = make_rsrc(static_cast<const T*>(a.q) + ((int64_t)sp.q0 + j0) * a.q_ld + (int64_t)hk * group * a.q_hd, 0x7fffffff);
      const int here = (int)min(rows - (int64_t)at * 64, (int64_t)64);
#pragma unroll
      for (int i = 0; i < S::IT; ++i)
        st.held[i] = __builtin_amdgcn_raw_buffer_load_b128(rq, S::row(i) < here ? off[i] : kOOB, 0, 0);
      if (threadIdx.x < 64) {
        lim = 0;
        rl = make_float2(0.f, 1.f);
        if ((int)threadIdx.x < here) {
          lim = visible(sp, j0 + sj, a.causal);
          const int64_t id = ((int64_t)sp.q0 + j0 + sj) * a.heads + hk * group + sh;
          rl = a.rl[id];                     // (of all parts: see rows_body)
        }
      }
      ++at;
      j0 += step;
      rem += left;
      if (left) {
        if (rem >= group) rem -= group, ++j0;
        places();
      }
    };
    auto put = [&](int buf) {
      st.put(tile[buf]);
      if (threadIdx.x < 64) stat[buf][threadIdx.x] = (f32x4_t){rl.x, share(rl.y, lim), u.unit(rl.x), __int_as_float(lim)};
    };
    __syncthreads();                          // the last keys' tiles are read
    if (tb < te) {
      load();
      put(0);
      if (tb + 1 < te) load();
      __syncthreads();
      int buf = 0;
      int t = tb;
      // Tiles up to `end`.  Two bodies in one loop would move the sums between registers at each tile.
      auto pass = [&](auto masked, int end) {
        for (; t < end; ++t, buf ^= 1) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            f32x16_t s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
            const int q = m * 32 + l32, z = Lds<T, D>::kswz(q);
            const T* base = tile[buf] + q * D;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              G qf;
              if constexpr (sizeof(T) == 2) {
                qf.v = *reinterpret_cast<const u32x4_t*>(base + ((2 * i + hh) ^ z) * S::PER);
              } else {
                qf.lo = *reinterpret_cast<const u32x4_t*>(base + ((4 * i + 2 * hh) ^ z) * S::PER);
                qf.hi = *reinterpret_cast<const u32x4_t*>(base + ((4 * i + 2 * hh + 1) ^ z) * S::PER);
              }
              s = mfma32_k16(kr[i], qf, s);
            }
            const f32x4_t c = stat[buf][q];
            const int room = __float_as_int(c[3]) - kc - hh * 4;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c[2], -c[0]));
              if constexpr (decltype(masked)::value) sum[r] += (r >> 2) * 8 + (r & 3) < room ? e * c[1] : 0.f;
              else sum[r] = __builtin_fmaf(e, c[1], sum[r]);
            }
          }
          if (t + 1 < te) put(buf ^ 1);
          if (t + 2 < te) load();
          __syncthreads();
        }
      };
      // from which tile on every row sees all of the workgroup's keys, up to the last tile that is whole
      const int64_t from = a.causal ? min(k0 + 128, (int64_t)sp.k_lim) - 1 - ((int64_t)sp.k_len - sp.q_len) : 0;
      const int full0 = (int)(min(max(from, (int64_t)0) * group + 63, rows) >> 6), full1 = min((int)(rows >> 6), te);
      pass(std::true_type{}, min(full0, te));
      pass(std::false_type{}, full1);
      pass(std::true_type{}, te);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) sum[r] += __shfl_xor(sum[r], m);
    }
    if (l32 == 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kc + (r >> 2) * 8 + hh * 4 + (r & 3);
        if (key >= sp.k_lim) continue;
        if (parts > 1) {
          a.scores[((int64_t)part * a.s.n * a.kv + pair) * a.s_ld + key] = sum[r];
        } else {
          float* to = acc + (int64_t)key * a.acc_ld;
          *to = (a.decay == 0.f ? 0.f : a.decay * *to) + sum[r];
        }
      }
    }
  }
}

// The parts of the rows, joined in order.
__device__ __forceinline__ void join_body(const vrs_weights_args& a) {
  const int pair = blockIdx.x, hk = pair % a.kv;
  const SeqSpan sp = seq_span(a.s, pair / a.kv);
  const int64_t key = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (key >= sp.k_lim || key >= a.s_ld) return;
  float* to = a.acc + (sp.k0 + key) * a.acc_ld + hk * a.acc_hd;
  const float old = a.decay == 0.f ? 0.f : a.decay * *to;
  float sum = 0.f;
#pragma unroll 4
  for (int p = 0; p < a.key_parts; ++p) sum += a.scores[((int64_t)p * a.s.n * a.kv + pair) * a.s_ld + key];
  *to = old + sum;
}
}  // namespace

#define VRS_WEIGHTS(TN, T, D, WPS)                                                                                                 \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_weights_scores_##TN##_d##D(vrs_weights_args a) { scores_body<T, D>(a); } \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_weights_stats_##TN##_d##D(vrs_weights_args a) { stats_body<T, D>(a); } \
  extern "C" __global__ __launch_bounds__(256, WPS) void vrs_weights_keys_##TN##_d##D(vrs_weights_args a) { keys_body<T, D>(a); }
VRS_WEIGHTS(bf16, bf16_t, 64, 3)
VRS_WEIGHTS(bf16, bf16_t, 128, 3)
VRS_WEIGHTS(f32, float, 64, 2)
VRS_WEIGHTS(f32, float, 128, 1)
extern "C" __global__ __launch_bounds__(256) void vrs_weights_sum_bf16(vrs_weights_args a) { sum_body<bf16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_weights_sum_f32(vrs_weights_args a) { sum_body<float>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_weights_rows(vrs_weights_args a) { rows_body(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_weights_join(vrs_weights_args a) { join_body(a); }
