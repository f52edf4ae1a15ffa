// Rotary positions for gfx950: pairs (a, b) of each head turn by an angle
// that grows with the row's position,
//   (a, b) -> scale * (a cos t - b sin t, a sin t + b cos t),  t = 2 pi pos freq[i]
// the same for every head, so a row's cosines and sines are computed once
// (position times frequency in 64 bits, of which the fraction of a turn goes
// to float32: exact for any 32-bit position) and read from LDS by all heads.
//
// Memory bound: q, k (and v on its way into a cache) read and written once.
// WPR waves take a row: they load q's first vectors, compute the row's angles
// into LDS meanwhile, then walk its heads, kBatch vectors (or pairs of them) of
// a thread at a time, all of a batch's loads before its stores.  Many rows: a
// wave to a row, no barrier.  7283 rows of 32 + 8 heads of 128 and 8 of values
// into a cache in bfloat16, 179 MB: 38 us, 4.7 TB/s (42 us with the angles
// first and a barrier for four rows).
#include "seqs.h"

namespace {
// VEC elements as they lie in memory: 16 bytes, 8, or one element.
template <typename T, int VEC>
struct Vec {
  typedef uint32_t U __attribute__((ext_vector_type(VEC * sizeof(T) / 4)));
  U u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const U*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<U*>(p) = u; }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
    else return __uint_as_float((i & 1) ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < (int)(VEC * sizeof(T) / 4); ++i) {
      if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(f[i]);
      else u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
  }
};
template <typename T>
struct Vec<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ float operator[](int) const { return Elt<T>::to_f(v); }
  __device__ __forceinline__ void set(const float* f) { v = Elt<T>::from_f(f[0]); }
};

constexpr int kMaxPairs = 256, kBatch = 4;

// The turned part of a row's heads: `per` items of VEC pairs to a head, a
// thread's items NT apart, kBatch of them from j0 on at a time.  Items past
// the last load that one again, so that no load sits behind a branch.
template <typename T, int VEC, int NT>
struct Turn {
  Vec<T, VEC> x[kBatch], y[kBatch];
  int head[kBatch], e0[kBatch], w[kBatch];
  int n, per, step;
  float inv;
  bool pairs;

  __device__ __forceinline__ Turn(int heads, int per_, int half, bool pairs_) {
    per = per_;
    n = heads * per;
    inv = 1.f / (float)per;
    pairs = pairs_;
    step = pairs ? VEC : half;                  // from an item's first vector to its second
  }
  __device__ __forceinline__ void load(int j0, const T* src, int64_t hd) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      int c;
      head[b] = fdivmod(min(j0 + b * NT, n - 1), per, inv, c);
      w[b] = c * VEC;                           // its first pair
      e0[b] = pairs ? 2 * w[b] : w[b];
      x[b].load(src + head[b] * hd + e0[b]);
      y[b].load(src + head[b] * hd + e0[b] + step);
    }
  }
  __device__ __forceinline__ void store(int j0, T* dst, int64_t hd, const float2* cs) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (j0 + b * NT >= n) break;
      float f[2 * VEC], o[2 * VEC];             // in the order of memory
#pragma unroll
      for (int p = 0; p < VEC; ++p) f[p] = x[b][p], f[VEC + p] = y[b][p];
#pragma unroll
      for (int p = 0; p < VEC; ++p) {
        const float2 c = cs[w[b] + p];
        const float va = pairs ? f[2 * p] : f[p], vb = pairs ? f[2 * p + 1] : f[VEC + p];
        const float oa = va * c.x - vb * c.y, ob = va * c.y + vb * c.x;
        // where the pair lies differs, what is written there does not depend on the other layout
        if (pairs) o[2 * p] = oa, o[2 * p + 1] = ob;
        else o[p] = oa, o[VEC + p] = ob;
      }
      x[b].set(o);
      y[b].set(o + VEC);
      T* to = dst + head[b] * hd + e0[b];
      x[b].store(to);
      y[b].store(to + step);
    }
  }
  // all items; the first batch may have been loaded already
  __device__ __forceinline__ void run(int t, bool loaded, const T* src, int64_t src_hd, T* dst, int64_t dst_hd,
                                      const float2* cs) {
    for (int j0 = t; j0 < n; j0 += kBatch * NT) {
      if (!loaded || j0 != t) load(j0, src, src_hd);
      store(j0, dst, dst_hd, cs);
    }
  }
};
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
      int c;
      head[b] = fdivmod(min(j0 + b * NT, n - 1), per, inv, c);
      e[b] = (from + c) * VEC;
      x[b].load(src + head[b] * src_hd + e[b]);
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
  const int half = a.rot / 2, pc = half / VEC, rc = a.rot / VEC, vc = a.dim / VEC;   // chunks of a head
  // q's first loads do not wait for the row's place and angles
  const T* q = static_cast<const T*>(a.q) + min(row, (int64_t)a.rows - 1) * a.q_ld;
  Turn<T, VEC, NT> turn(a.heads, pc, half, a.pairs_layout);
  if (a.heads) turn.load(t, q, a.q_hd);
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

  T* qo = static_cast<T*>(a.qo) + row * a.qo_ld;
  turn.run(t, true, q, a.q_hd, qo, a.qo_hd, cs);
  if (rc < vc && a.q != a.qo) copy_heads<T, VEC, NT>(q, a.q_hd, qo, a.qo_hd, a.heads, rc, vc - rc, t);
  if (to < 0 || a.kv == 0) return;
  const T* k = static_cast<const T*>(a.k) + row * a.k_ld;
  T* ko = static_cast<T*>(a.ko) + to * a.ko_ld;
  Turn<T, VEC, NT>(a.kv, pc, half, a.pairs_layout).run(t, false, k, a.k_hd, ko, a.ko_hd, cs);
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
