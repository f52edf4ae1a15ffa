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

// Stage 1: a workgroup of 4 waves takes 32 rows of one key head against a part of
// the keys, its waves every fourth 32 of them.
template <typename T, int D, bool KEEP>
__device__ __forceinline__ void stats_body(const vrs_weights_args& a) {
  using E = Elt<T>;
  using G = typename E::group;
  constexpr int NW = 4;
  __shared__ float sR[NW][32], sl[NW][32];
  const int wave = threadIdx.x >> 6;
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
    G kr[D / 16];
    uint32_t ko[D / 16];                   // offsets in a tile; elements past the head read 0
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = i * 16 + w.hh * 8;
      ko[i] = d < a.dim ? (uint32_t)(w.l32 * (int)a.k_ld + d) * (uint32_t)sizeof(T) : kOOB;
    }
    auto load = [&](int kc) {              // keys past the sequence's last are masked, whatever they read
      const int n = min(32, sp.k_lim - kc);
      const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) kr[i] = E::bload(rk, ko[i], 0);
    };
    float* keep = a.scores + (row * a.heads + h) * a.s_ld;
    int kc = kb + wave * 32;
    if (kc < ke) load(kc);
    while (kc < ke) {
      f32x16_t s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s = mfma32_k16(kr[i], w.qf[0][i], s);
      const int at = kc;
      kc += NW * 32;
      if (kc < ke) load(kc);
      if (at + 32 > lim_min) w.mask(0, s, at);
      if constexpr (KEEP) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int64_t key = at + g * 8 + w.hh * 4;
          const f32x4_t v = {s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
          if (ok && key < a.s_ld) *reinterpret_cast<f32x4_t*>(keep + key) = v;
        }
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

// A row's reference and 1 / sum over the parts of its keys.
__device__ __forceinline__ float2 joined(const vrs_weights_args& a, const Log2& u, int64_t id, int keys) {
  const int64_t step = (int64_t)a.s.q_rows * a.heads;
  float mx = kNone, l = 0.f;
  for (int p = 0; p < a.parts; ++p) mx = fmaxf(mx, a.rl[p * step + id].x);
  for (int p = 0; p < a.parts; ++p) {
    const float2 rl = a.rl[p * step + id];
    l += u.factor(rl.x, mx) * rl.y;
  }
  return make_float2(mx, share(l, keys));
}

// Stage 2 from the scores: a thread takes a key and passes over the rows.
template <typename T>
__device__ __forceinline__ void sum_body(const vrs_weights_args& a) {
  constexpr int RB = 64;
  __shared__ float sR[RB], sinv[RB], sunit[RB];
  __shared__ int slim[RB];
  const int hk = blockIdx.x % a.kv;
  const SeqSpan sp = seq_span(a.s, blockIdx.x / a.kv);
  const int G_ = a.heads / a.kv;
  const int rows = (int)min((int64_t)sp.q_len * G_, (int64_t)0x7fffffff);
  const Log2 u(a.c);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  float* acc = a.acc + sp.k0 * a.acc_ld + hk * a.acc_hd;
  for (int64_t k0 = (int64_t)blockIdx.y * 256; k0 < sp.k_lim; k0 += (int64_t)gridDim.y * 256) {
    const int key = (int)k0 + threadIdx.x;
    float sum = 0.f;
    for (int r0 = 0; r0 < rows; r0 += RB) {
      __syncthreads();
      const int r = r0 + threadIdx.x;
      if (threadIdx.x < RB && r < rows) {
        const int j = r / G_;
        const int64_t id = ((int64_t)sp.q0 + j) * a.heads + hk * G_ + (r - j * G_);
        const int lim = visible(sp, j, a.causal);
        const float2 rl = joined(a, u, id, lim);
        sR[threadIdx.x] = rl.x;
        sinv[threadIdx.x] = rl.y;
        sunit[threadIdx.x] = u.unit(rl.x);
        slim[threadIdx.x] = lim;
      }
      __syncthreads();
      if (key < sp.k_lim) {
        for (int i = 0; i < min(RB, rows - r0); ++i) {
          if (key >= slim[i]) continue;
          const int j = (r0 + i) / G_, h = hk * G_ + (r0 + i - j * G_);
          const int64_t row = (int64_t)sp.q0 + j;
          float s;
          if (key < a.s_ld) {
            s = a.scores[(row * a.heads + h) * a.s_ld + key];
          } else {                         // more keys than were counted on
            const T* q = static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd;
            const T* k = kp + (int64_t)key * a.k_ld;
            s = 0.f;
            for (int d = 0; d < a.dim; ++d) s = __builtin_fmaf(Elt<T>::to_f(q[d]), Elt<T>::to_f(k[d]), s);
          }
          sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s, sunit[i], -sR[i])) * sinv[i];
        }
      }
    }
    if (key < sp.k_lim) {
      float* to = acc + (int64_t)key * a.acc_ld;
      *to = (a.decay == 0.f ? 0.f : a.decay * *to) + sum;
    }
  }
}

// Stage 2 with the products again: a wave holds 32 keys, and the rows that see
// them pass by in tiles of 32.
template <typename T, int D>
__device__ __forceinline__ void keys_body(const vrs_weights_args& a) {
  using E = Elt<T>;
  using G = typename E::group;
  const int hk = blockIdx.x % a.kv, wave = threadIdx.x >> 6, l32 = threadIdx.x & 31, hh = (threadIdx.x >> 5) & 1;
  const SeqSpan sp = ranked_seq(Sequences{a.s}, blockIdx.x / a.kv);
  const int G_ = a.heads / a.kv;
  const int64_t rows = (int64_t)sp.q_len * G_;
  const Log2 u(a.c);
  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  float* acc = a.acc + sp.k0 * a.acc_ld + hk * a.acc_hd;
  for (int64_t k0 = (int64_t)blockIdx.y * 128 + wave * 32; k0 < sp.k_lim; k0 += (int64_t)gridDim.y * 128) {
    const int kc = (int)k0;
    G kr[D / 16];
    const int n = min(32, sp.k_lim - kc);
    const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = i * 16 + hh * 8;
      kr[i] = E::bload(rk, d < a.dim ? (uint32_t)(l32 * (int)a.k_ld + d) * (uint32_t)sizeof(T) : kOOB, 0);
    }
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    // rows from the first that sees key kc on
    const int64_t skip = a.causal ? max((int64_t)0, (int64_t)kc - ((int64_t)sp.k_len - sp.q_len)) * G_ : 0;
    for (int64_t r0 = skip / 32 * 32; r0 < rows; r0 += 32) {
      const int64_t pr = min(r0 + l32, rows - 1);
      const bool ok = r0 + l32 < rows;
      const int j = (int)(pr / G_), h = hk * G_ + (int)(pr - (int64_t)j * G_);
      const int64_t row = sp.q0 + j;
      const int lim = ok ? visible(sp, j, a.causal) : 0;
      const T* q = static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd;
      const float2 rl = joined(a, u, row * a.heads + h, lim);
      const float unit = u.unit(rl.x);
      f32x16_t s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const int d = i * 16 + hh * 8;
        s = mfma32_k16(kr[i], d < a.dim ? E::load(q + d) : E::zero(), s);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = kc + (r >> 2) * 8 + hh * 4 + (r & 3);
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], unit, -rl.x)) * rl.y;
        sum[r] += key < lim ? p : 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) sum[r] += __shfl_xor(sum[r], m);
      const int key = kc + (r >> 2) * 8 + hh * 4 + (r & 3);
      if (l32 == 0 && key < sp.k_lim) {
        float* to = acc + (int64_t)key * a.acc_ld;
        *to = (a.decay == 0.f ? 0.f : a.decay * *to) + sum[r];
      }
    }
  }
}
}  // namespace

#define VRS_WEIGHTS(TN, T, D)                                                                                                 \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_weights_scores_##TN##_d##D(vrs_weights_args a) { stats_body<T, D, true>(a); } \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_weights_stats_##TN##_d##D(vrs_weights_args a) { stats_body<T, D, false>(a); } \
  extern "C" __global__ __launch_bounds__(256, 2) void vrs_weights_keys_##TN##_d##D(vrs_weights_args a) { keys_body<T, D>(a); }
VRS_WEIGHTS(bf16, bf16_t, 64)
VRS_WEIGHTS(bf16, bf16_t, 128)
VRS_WEIGHTS(f32, float, 64)
VRS_WEIGHTS(f32, float, 128)
extern "C" __global__ __launch_bounds__(256) void vrs_weights_sum_bf16(vrs_weights_args a) { sum_body<bf16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_weights_sum_f32(vrs_weights_args a) { sum_body<float>(a); }
