// Rotary positions for gfx950: pairs (a, b) of each head turn by an angle
// that grows with the row's position,
//   (a, b) -> scale * (a cos t - b sin t, a sin t + b cos t),  t = 2 pi pos freq[i]
// the same for every head, so a row's cosines and sines are computed once
// (position times frequency in 64 bits, of which the fraction of a turn goes
// to float32: exact for any 32-bit position) and read from LDS by all heads.
//
// Memory bound: q, k (and v on its way into a cache) read and written once.
// WPR waves take a row: they compute its angles into LDS, then walk its heads,
// kBatch vectors (or pairs of them) of a thread at a time, all of a batch's
// loads before its stores.  Many rows: a wave to a row, no barrier.
#include "seqs.h"

namespace {
template <typename T, int VEC>
struct Vec {
  float f[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      f[0] = Elt<T>::to_f(*p);
    } else {
      typedef uint32_t U __attribute__((ext_vector_type(VEC * sizeof(T) / 4)));
      const U u = *reinterpret_cast<const U*>(p);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(u[i]);
        else f[i] = __uint_as_float((i & 1) ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC == 1) {
      *p = Elt<T>::from_f(f[0]);
    } else {
      typedef uint32_t U __attribute__((ext_vector_type(VEC * sizeof(T) / 4)));
      U u;
#pragma unroll
      for (int i = 0; i < (int)(VEC * sizeof(T) / 4); ++i) {
        if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(f[i]);
        else u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      }
      *reinterpret_cast<U*>(p) = u;
    }
  }
};

constexpr int kMaxPairs = 256, kBatch = 4;

// The turned part of a row's heads: `per` items of VEC pairs to a head, threads t, t + NT, ...
template <typename T, int VEC, int NT>
__device__ __forceinline__ void turn_heads(const T* src, int64_t src_hd, T* dst, int64_t dst_hd, int heads, int per,
                                           int half, bool pairs, const float2* cs, int t) {
  const float inv = 1.f / (float)per;
  const int n = heads * per;
  for (int j0 = t; j0 < n; j0 += kBatch * NT) {
    Vec<T, VEC> x[kBatch], y[kBatch];
    int head[kBatch], e0[kBatch], w[kBatch];
    const int step = pairs ? VEC : half;        // from an item's first vector to its second
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = j0 + b * NT;
      int c;
      head[b] = fdivmod(min(j, n - 1), per, inv, c);
      w[b] = c * VEC;                           // its first pair
      e0[b] = pairs ? 2 * w[b] : w[b];
      if (j < n) {
        x[b].load(src + head[b] * src_hd + e0[b]);
        y[b].load(src + head[b] * src_hd + e0[b] + step);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (j0 + b * NT >= n) break;
      float f[2 * VEC];                         // in the order of memory
#pragma unroll
      for (int p = 0; p < VEC; ++p) f[p] = x[b].f[p], f[VEC + p] = y[b].f[p];
#pragma unroll
      for (int p = 0; p < VEC; ++p) {
        const float2 c = cs[w[b] + p];
        const float ha = f[p], hb = f[VEC + p], pa = f[2 * p], pb = f[2 * p + 1];
        const float va = pairs ? pa : ha, vb = pairs ? pb : hb;
        const float oa = va * c.x - vb * c.y, ob = va * c.y + vb * c.x;
        if (pairs) {
          if (2 * p < VEC) x[b].f[(2 * p) % VEC] = oa;
          else y[b].f[(2 * p) % VEC] = oa;
          if (2 * p + 1 < VEC) x[b].f[(2 * p + 1) % VEC] = ob;
          else y[b].f[(2 * p + 1) % VEC] = ob;
        } else {
          x[b].f[p] = oa;
          y[b].f[p] = ob;
        }
      }
      T* to = dst + head[b] * dst_hd + e0[b];
      x[b].store(to);
      y[b].store(to + step);
    }
  }
}
// The vectors [from, from + per) of a row's heads as they are.
template <typename T, int VEC, int NT>
__device__ __forceinline__ void copy_heads(const T* src, int64_t src_hd, T* dst, int64_t dst_hd, int heads, int from,
                                           int per, int t) {
  const float inv = 1.f / (float)per;
  const int n = heads * per;
  for (int j0 = t; j0 < n; j0 += kBatch * NT) {
    Vec<T, VEC> x[kBatch];
    int head[kBatch], e[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = j0 + b * NT;
      int c;
      head[b] = fdivmod(min(j, n - 1), per, inv, c);
      e[b] = (from + c) * VEC;
      if (j < n) x[b].load(src + head[b] * src_hd + e[b]);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (j0 + b * NT < n) x[b].store(dst + head[b] * dst_hd + e[b]);
  }
}

template <typename T, int VEC, int WPR>
__device__ __forceinline__ void rope_body(const vrs_rope_args& a) {
  constexpr int RPW = 4 / WPR, NT = WPR * 64;        // rows of a workgroup, threads of a row
  __shared__ float2 angles[RPW][kMaxPairs];
  const int r = __builtin_amdgcn_readfirstlane(threadIdx.x / NT), t = threadIdx.x % NT;
  const int64_t row = (int64_t)blockIdx.x * RPW + r;
  float2* cs = angles[r];
  const int half = a.rot / 2;
  bool ok = row < a.rows;              // whether the row is a sequence's
  int64_t to = ok ? row : -1;          // where its k and v go; -1: nowhere
  int place = (int)row;
  if (ok && a.s.q_start) {
    ok = row >= a.s.q_start[0];
    if (ok) {
      const int i = find_seq(a.s.n, (int)row, [&](int j) { return a.s.q_start[j]; });
      const SeqSpan sp = seq_span(a.s, i);
      ok = row >= sp.q0 && row < sp.q0 + sp.q_len;
      place = sp.k_len - sp.q_len + (int)(row - sp.q0);
      to = place >= 0 && place < sp.k_lim ? sp.k0 + place : -1;
    }
  }
  if (ok) {
    for (int i = t; i < half; i += NT) {
      int p = place;
      if (a.pos) {
        const int ax = (i >= a.axis_end[0]) + (i >= a.axis_end[1]) + (i >= a.axis_end[2]);
        p = a.pos[ax * a.pos_ld + row];
      }
      double turns = (double)p * a.freq[i];
      turns -= rint(turns);
      float sn, cn;
      sincospif(2.f * (float)turns, &sn, &cn);
      cs[i] = make_float2(cn * a.scale, sn * a.scale);
    }
  }
  if constexpr (WPR > 1) __syncthreads();
  else __builtin_amdgcn_wave_barrier();        // one wave's LDS: order alone is needed
  if (!ok) return;

  const int pc = half / VEC, rc = a.rot / VEC, vc = a.dim / VEC;   // chunks of a head
  const T* q = static_cast<const T*>(a.q) + row * a.q_ld;
  T* qo = static_cast<T*>(a.qo) + row * a.qo_ld;
  turn_heads<T, VEC, NT>(q, a.q_hd, qo, a.qo_hd, a.heads, pc, half, a.pairs_layout, cs, t);
  if (rc < vc && a.q != a.qo) copy_heads<T, VEC, NT>(q, a.q_hd, qo, a.qo_hd, a.heads, rc, vc - rc, t);
  if (to < 0 || a.kv == 0) return;
  const T* k = static_cast<const T*>(a.k) + row * a.k_ld;
  T* ko = static_cast<T*>(a.ko) + to * a.ko_ld;
  turn_heads<T, VEC, NT>(k, a.k_hd, ko, a.ko_hd, a.kv, pc, half, a.pairs_layout, cs, t);
  if (rc < vc && a.k != a.ko) copy_heads<T, VEC, NT>(k, a.k_hd, ko, a.ko_hd, a.kv, rc, vc - rc, t);
  if (a.v)
    copy_heads<T, VEC, NT>(static_cast<const T*>(a.v) + row * a.v_ld, a.v_hd, static_cast<T*>(a.vo) + to * a.vo_ld, a.vo_hd,
                           a.kv, 0, vc, t);
}
}  // namespace

#define VRS_ROPE(TN, T, VEC, WPR)                                                                      \
  extern "C" __global__ __launch_bounds__(256) void vrs_rope_##TN##_v##VEC##_w##WPR(vrs_rope_args a) { \
    rope_body<T, VEC, WPR>(a);                                                                         \
  }
VRS_ROPE(bf16, bf16_t, 8, 1)
VRS_ROPE(bf16, bf16_t, 8, 4)
VRS_ROPE(bf16, bf16_t, 4, 1)
VRS_ROPE(bf16, bf16_t, 4, 4)
VRS_ROPE(bf16, bf16_t, 1, 1)
VRS_ROPE(bf16, bf16_t, 1, 4)
VRS_ROPE(f32, float, 4, 1)
VRS_ROPE(f32, float, 4, 4)
VRS_ROPE(f32, float, 1, 1)
VRS_ROPE(f32, float, 1, 4)
