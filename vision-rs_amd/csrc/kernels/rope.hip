// Rotary positions for gfx950: pairs (a, b) of each head turn by an angle
// that grows with the row's position,
//   (a, b) -> scale * (a cos t - b sin t, a sin t + b cos t),  t = 2 pi pos freq[i]
// the same for every head, so a row's cosines and sines are computed once
// (position times frequency in 64 bits, of which the fraction of a turn goes
// to float32: exact for any 32-bit position) and read from LDS by all heads.
//
// Memory bound: q, k (and v on its way into a cache) read and written once.
// A workgroup takes RPW rows, one wave computing the angles of each; its
// threads then walk the rows' items: VEC pairs, or a vector that is only
// copied (the part of a head past rot, and v).
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

constexpr int kMaxPairs = 256;

template <typename T, int VEC, int RPW>
__device__ __forceinline__ void rope_body(const vrs_rope_args& a) {
  __shared__ float2 cs[RPW][kMaxPairs];
  __shared__ int64_t key_row[RPW];     // where the row's k and v go; -1: nowhere
  __shared__ int live[RPW];
  const int half = a.rot / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * RPW;
  for (int r = wave; r < RPW; r += 4) {
    const int64_t row = row0 + r;
    bool ok = row < a.rows;
    int64_t to = ok ? row : -1;
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
    if (lane == 0) {
      live[r] = ok;
      key_row[r] = to;
    }
    if (ok) {
      for (int i = lane; i < half; i += 64) {
        int p = place;
        if (a.pos) {
          int ax = 0;
          while (ax + 1 < a.axes && i >= a.axis_end[ax]) ++ax;
          p = a.pos[ax * a.pos_ld + row];
        }
        double t = (double)p * a.freq[i];
        t -= rint(t);
        float sn, cn;
        sincospif(2.f * (float)t, &sn, &cn);
        cs[r][i] = make_float2(cn * a.scale, sn * a.scale);
      }
    }
  }
  __syncthreads();
  const int pc = half / VEC, tc = (a.dim - a.rot) / VEC, vc = a.dim / VEC;   // chunks of a head
  for (int it = threadIdx.x; it < RPW * a.items; it += 256) {
    int j;
    const int r = fdivmod(it, a.items, a.inv_items, j);
    if (!live[r]) continue;
    const int64_t row = row0 + r;
    const T* src;
    T* dst;
    bool turn = false;
    int c;
    if (j < a.qi + a.qt) {
      const int per = j < a.qi ? pc : tc;
      turn = j < a.qi;
      if (!turn) j -= a.qi;
      const int h = j / per;
      c = turn ? j - h * per : a.rot / VEC + j - h * per;
      src = static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd;
      dst = static_cast<T*>(a.qo) + row * a.qo_ld + h * a.qo_hd;
    } else {
      j -= a.qi + a.qt;
      const int64_t to = key_row[r];
      if (to < 0) continue;
      if (j < a.ki + a.kt) {
        const int per = j < a.ki ? pc : tc;
        turn = j < a.ki;
        if (!turn) j -= a.ki;
        const int h = j / per;
        c = turn ? j - h * per : a.rot / VEC + j - h * per;
        src = static_cast<const T*>(a.k) + row * a.k_ld + h * a.k_hd;
        dst = static_cast<T*>(a.ko) + to * a.ko_ld + h * a.ko_hd;
      } else {
        j -= a.ki + a.kt;
        const int h = j / vc;
        c = j - h * vc;
        src = static_cast<const T*>(a.v) + row * a.v_ld + h * a.v_hd;
        dst = static_cast<T*>(a.vo) + to * a.vo_ld + h * a.vo_hd;
      }
    }
    Vec<T, VEC> x, y;
    if (!turn) {
      x.load(src + c * VEC);
      x.store(dst + c * VEC);
      continue;
    }
    const int e0 = a.pairs_layout ? 2 * c * VEC : c * VEC;
    const int e1 = a.pairs_layout ? e0 + VEC : half + c * VEC;
    x.load(src + e0);
    y.load(src + e1);
    Vec<T, VEC> ox, oy;
#pragma unroll
    for (int p = 0; p < VEC; ++p) {
      const float2 w = cs[r][c * VEC + p];
      if (a.pairs_layout) {     // pair p: elements 2p, 2p + 1 of the two vectors
        float va, vb;
        if constexpr (VEC == 1) va = x.f[0], vb = y.f[0];
        else va = 2 * p < VEC ? x.f[(2 * p) % VEC] : y.f[(2 * p) % VEC],
             vb = 2 * p < VEC ? x.f[(2 * p + 1) % VEC] : y.f[(2 * p + 1) % VEC];
        const float oa = va * w.x - vb * w.y, ob = va * w.y + vb * w.x;
        if constexpr (VEC == 1) ox.f[0] = oa, oy.f[0] = ob;
        else if (2 * p < VEC) ox.f[(2 * p) % VEC] = oa, ox.f[(2 * p + 1) % VEC] = ob;
        else oy.f[(2 * p) % VEC] = oa, oy.f[(2 * p + 1) % VEC] = ob;
      } else {
        ox.f[p] = x.f[p] * w.x - y.f[p] * w.y;
        oy.f[p] = x.f[p] * w.y + y.f[p] * w.x;
      }
    }
    ox.store(dst + e0);
    oy.store(dst + e1);
  }
}
}  // namespace

#define VRS_ROPE(TN, T, VEC, RPW)                                                                         \
  extern "C" __global__ __launch_bounds__(256) void vrs_rope_##TN##_v##VEC##_r##RPW(vrs_rope_args a) { \
    rope_body<T, VEC, RPW>(a);                                                                            \
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
