// Beam search's step, for gfx950: the selection of the best continuations over a
// request's beams and vocabulary, and the reordering of the beams' states.
//
// Selection, c_it = s_i + (x_it - lse_i), in two launches.  First a workgroup takes
// a chunk of one row of logits into registers, in one pass over memory: its maximum
// and sum of exp, and its k largest logits in order.  Then a workgroup joins the
// chunks of a request: the rows' lse, and the k largest of what the chunks left.
//
// The k largest of a workgroup's numbers: the r-th largest of a wave's lane maxima,
// r = k / waves, is reached by k numbers at least, and by few more where their order
// is that of a vocabulary.  Those that reach it go to LDS and each counts how many
// beat it, which is its place.  Where they are too many (equal or sorted logits) the
// workgroup takes its maximum k times instead.
#include "common.h"

namespace {
constexpr int kT = 256, kWaves = kT / 64;
constexpr int kCand = 1024;                  // candidates that LDS holds

// Order of floats and doubles as whole numbers (both zeros alike is the caller's)
__device__ __forceinline__ uint32_t order32(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order64(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}

// A number that r lanes of the wave reach at least, within 2^-15 of the r-th largest one's order (0: no number).
__device__ __forceinline__ uint32_t reached(uint32_t o, int r) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 12; --b) {
    const uint32_t trial = t | 1u << b;
    if (__builtin_popcountll(__ballot(o >= trial)) >= r) t = trial;
  }
  return t;
}

// Maximum over the workgroup of (order, -place): the lowest place of the largest.
__device__ __forceinline__ void best_of(uint64_t& o, uint32_t& at, uint64_t (&so)[kWaves], uint32_t (&sat)[kWaves]) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t p = (uint64_t)__shfl_xor((unsigned long long)o, m);
    const uint32_t q = __shfl_xor(at, m);
    if (p > o || (p == o && q < at)) o = p, at = q;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) so[threadIdx.x >> 6] = o, sat[threadIdx.x >> 6] = at;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    if (so[w] > o || (so[w] == o && sat[w] < at)) o = so[w], at = sat[w];
}

// ---------------------------------------------------------------------------
// A chunk of one row: VT vectors of 16 bytes to a thread.
template <typename T, int VT>
__device__ __forceinline__ void part_body(const vrs_beam_args& a) {
  constexpr int V = 16 / (int)sizeof(T), N = VT * V;
  __shared__ uint2 cand[kCand];
  __shared__ int count;
  __shared__ float swm[kWaves];
  __shared__ double sws[kWaves];
  __shared__ uint32_t sth[kWaves], salone[kWaves];
  __shared__ uint64_t so[kWaves];
  __shared__ uint32_t sat[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int ch = blockIdx.x, row = blockIdx.y;
  if (a.done && a.done[row]) return;           // such a beam goes on with the end token alone
  const int c0 = ch * a.chunk, n = min(a.chunk, a.vocab - c0);
  const T* x = static_cast<const T*>(a.logits) + (int64_t)row * a.ld + c0;
  float v[N];
  bool nan = false;
#pragma unroll
  for (int j = 0; j < VT; ++j) {
    const int e0 = (j * kT + tid) * V;
    if (e0 + V <= n) {
      T r[V];
      __builtin_memcpy(r, x + e0, 16);         // rows start anywhere
#pragma unroll
      for (int e = 0; e < V; ++e) v[j * V + e] = Elt<T>::to_f(r[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[j * V + e] = e0 + e < n ? Elt<T>::to_f(x[e0 + e]) : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    nan |= v[i] != v[i];
    m = fmaxf(m, v[i]);                        // (a NaN is passed over)
  }
  const float mine = m;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
  if (lane == 0) swm[wave] = m;
  // what every wave has at least ceil(k / waves) numbers of, or one of them k (short chunks fill one wave only)
  const uint32_t top = mine == -INFINITY ? 0 : order32(mine);
  const uint32_t each = reached(top, (a.k + kWaves - 1) / kWaves), alone = a.k <= 64 ? reached(top, a.k) : 0;
  if (lane == 0) sth[wave] = each, salone[wave] = alone;
  if (tid == 0) count = 0;
  __syncthreads();
  m = swm[0];
  uint32_t T0 = sth[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, swm[w]), T0 = min(T0, sth[w]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) T0 = max(T0, salone[w]);
  // the sum: 2^((x - m) log2 e), the exponent's factor in two parts, so that its rounding is that of one product
  float sum = 0.f;
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = v[i] - ref;
    sum += __builtin_amdgcn_exp2f(__builtin_fmaf(d, 1.44269502f, d * 1.92596300e-8f));
  }
  double total = nan ? (double)NAN : (double)sum;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) total += __shfl_xor(total, k);
  if (lane == 0) sws[wave] = total;
  // candidates
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = v[i] > -INFINITY && order32(v[i]) >= T0;      // (false for NaN)
    const uint64_t mask = __ballot(in);
    if (mask == 0) continue;
    int base = 0;
    if (lane == 0) base = atomicAdd(&count, __builtin_popcountll(mask));
    base = __builtin_amdgcn_readfirstlane(base) + __builtin_popcountll(mask & ((1ull << lane) - 1));
    if (in && base < kCand) cand[base] = make_uint2(order32(v[i]), (uint32_t)(c0 + ((i / V) * kT + tid) * V + i % V));
  }
  __syncthreads();
  const int64_t at = (int64_t)row * a.chunks + ch;
  if (tid == 0) a.part[at] = make_double2(m, sws[0] + sws[1] + sws[2] + sws[3]);
  uint2* list = a.list + at * a.k;
  const int have = count;
  auto logit = [](uint32_t o) { return o ^ (((int32_t)o >> 31) ? 0x80000000u : 0xffffffffu); };
  if (have <= kCand) {
    for (int i = tid; i < have; i += kT) {
      const uint2 me = cand[i];
      int rank = 0;
      for (int j = 0; j < have; ++j) rank += cand[j].x > me.x || (cand[j].x == me.x && cand[j].y < me.y);
      if (rank < a.k) list[rank] = make_uint2(logit(me.x), me.y);
    }
    if (tid < a.k && tid >= have) list[tid] = make_uint2(0, 0xffffffffu);
  } else {
    uint64_t lo = ~0ull;
    uint32_t lat = 0;                          // the last one taken
    for (int k = 0; k < a.k; ++k) {
      uint64_t o = 0;
      uint32_t p = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t q = (uint32_t)(c0 + ((i / V) * kT + tid) * V + i % V);
        const uint64_t c = v[i] > -INFINITY ? order32(v[i]) : 0;
        const bool after = c < lo || (c == lo && q > lat);
        if (c && after && (c > o || (c == o && q < p))) o = c, p = q;
      }
      best_of(o, p, so, sat);
      if (tid == 0) list[k] = o ? make_uint2(logit((uint32_t)o), p) : make_uint2(0, 0xffffffffu);
      lo = o, lat = p;
    }
  }
}

// ---------------------------------------------------------------------------
// A request: the rows' lse, then the k best of the chunks' lists.
template <typename T>
__device__ __forceinline__ void join_body(const vrs_beam_args& a) {
  __shared__ double lse[64], score[64];
  __shared__ uint8_t kind[64];                 // 0: nothing but -infinity, 1: its lists, 2: the end token alone
  __shared__ uint64_t co[kCand];
  __shared__ uint32_t cat[kCand];
  __shared__ uint32_t smax[kT];
  __shared__ int count, found;
  __shared__ uint32_t sth;
  __shared__ uint64_t so[kWaves];
  __shared__ uint32_t sat[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  // lse of a beam: a wave over its chunks
  for (int i = wave; i < a.beams; i += kWaves) {
    const int64_t row = (int64_t)b * a.beams + i;
    const float s = a.scores[row];
    const bool fine = s - s == 0.f, done = a.done && a.done[row];
    float m = -INFINITY;
    double l = 0;
    bool odd = false;
    if (!done) {
      for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, (float)a.part[row * a.chunks + c].x);
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k));
      for (int c = lane; c < a.chunks; c += 64) {
        const double2 p = a.part[row * a.chunks + c];
        if (p.y != p.y) odd = true;
        else if (p.y > 0.0) l += p.y * exp(p.x - (double)m);
      }
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) l += __shfl_xor(l, k);
      odd = __any(odd);
    }
    if (lane == 0) {
      score[i] = s;
      lse[i] = (double)m + log(l);
      kind[i] = !fine ? 0 : done ? 2 : (odd || m == -INFINITY || m == INFINITY) ? 0 : 1;
    }
  }
  if (tid == 0) count = 0, found = 0;
  __syncthreads();
  // entry j of list l (a beam's chunk): its order (0: none) and flat place
  const int lists = a.beams * a.chunks;
  const uint2* base = a.list + (int64_t)b * lists * a.k;
  auto entry = [&](int l, int j, uint64_t& o, uint32_t& at) {
    const int i = l / a.chunks;
    o = 0;
    if (kind[i] == 1) {
      const uint2 e = base[(int64_t)l * a.k + j];
      if (e.y != 0xffffffffu) {
        o = order64(score[i] + ((double)__uint_as_float(e.x) - lse[i]));
        at = (uint32_t)(i * a.vocab) + e.y;
      }
    } else if (kind[i] == 2 && j == 0 && l == i * a.chunks) {
      o = order64(score[i]);
      at = (uint32_t)(i * a.vocab + a.eos);
    }
  };
  // Lists are in order, so the first `per` entries of a list are its largest: a thread takes every per-th from
  // one of them, and the k-th largest of the threads' first ones is reached by k entries at least.
  int per = 1;
  while (per * 2 * lists <= kT) per *= 2;
  uint32_t top = 0;
  for (int l = tid / per; l < lists; l += kT / per) {
    uint64_t o = 0;
    uint32_t at = 0;
    if (tid % per < a.k) entry(l, tid % per, o, at);
    top = max(top, (uint32_t)(o >> 32));
  }
  smax[tid] = top;
  if (tid == 0) sth = 0;
  __syncthreads();
  int rank = 0;
  for (int j = 0; j < kT; ++j) rank += smax[j] > top || (smax[j] == top && j < tid);
  if (rank == a.k - 1) sth = top;
  __syncthreads();
  const uint32_t T0 = max(sth, 1u);
  for (int l = tid / per; l < lists; l += kT / per) {
    for (int j = tid % per; j < a.k; j += per) {
      uint64_t o;
      uint32_t at = 0;
      entry(l, j, o, at);
      if ((uint32_t)(o >> 32) < T0) break;
      const int p = atomicAdd(&count, 1);
      if (p < kCand) co[p] = o, cat[p] = at;
    }
  }
  __syncthreads();
  const int have = count;
  auto put = [&](int k, uint64_t o, uint32_t at) {
    const uint64_t bits = o ^ (((int64_t)o >> 63) ? 0x8000000000000000ull : ~0ull);
    a.out_scores[(int64_t)b * a.k + k] = (float)__builtin_bit_cast(double, bits);
    a.out_parents[(int64_t)b * a.k + k] = (int32_t)(at / (uint32_t)a.vocab);
    a.out_tokens[(int64_t)b * a.k + k] = (int32_t)(at % (uint32_t)a.vocab);
  };
  int got = min(have, a.k);
  if (have <= kCand) {
    for (int i = tid; i < have; i += kT) {
      const uint64_t o = co[i];
      const uint32_t at = cat[i];
      int r = 0;
      for (int j = 0; j < have; ++j) r += co[j] > o || (co[j] == o && cat[j] < at);
      if (r < a.k) put(r, o, at);
    }
  } else {
    uint64_t lo = ~0ull;
    uint32_t lat = 0;
    for (int k = 0; k < a.k; ++k) {
      uint64_t o = 0;
      uint32_t p = 0xffffffffu;
      for (int l = tid / per; l < lists; l += kT / per)
        for (int j = tid % per; j < a.k; j += per) {
          uint64_t c;
          uint32_t q = 0;
          entry(l, j, c, q);
          if (c == 0) break;
          const bool after = c < lo || (c == lo && q > lat);
          if (after && (c > o || (c == o && q < p))) o = c, p = q;
        }
      best_of(o, p, so, sat);
      if (tid == 0) put(k, o, p);
      lo = o, lat = p;
    }
  }
  // fewer than k: the lowest places whose score is -infinity
  const int64_t all = (int64_t)a.beams * a.vocab;
  for (int64_t f0 = 0; got < a.k && f0 < all; f0 += kT) {
    const int64_t f = f0 + tid;
    bool none = false;
    if (f < all) {
      const int i = (int)(f / a.vocab), t = (int)(f - (int64_t)i * a.vocab);
      if (kind[i] == 0) none = true;
      else if (kind[i] == 2) none = t != a.eos;
      else none = Elt<T>::to_f(static_cast<const T*>(a.logits)[((int64_t)b * a.beams + i) * a.ld + t]) == -INFINITY;
    }
    const uint64_t mask = __ballot(none);
    __syncthreads();
    if (lane == 0) sat[wave] = __builtin_popcountll(mask);
    __syncthreads();
    int p = got;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) p += sat[w];
      got += sat[w];
    }
    p += __builtin_popcountll(mask & ((1ull << lane) - 1));
    if (none && p < a.k) put(p, order64(-INFINITY), (uint32_t)f);
  }
}

// ---------------------------------------------------------------------------
// state[b][i] = old state[b][parent[b][i]] in place.  A thread takes one vector of a
// row for all beams of a request: it reads those that others go on from, and then
// writes them to where they go; no other thread touches that vector.
template <typename V, int B>
__device__ __forceinline__ void reorder_body(const vrs_reorder_args& a) {
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  int parent = lane, len = a.rows;
  if (lane < a.beams) {
    const int p = a.parents[(int64_t)b * a.beams + lane];
    parent = p >= 0 && p < a.beams ? p : lane;
    if (a.len) len = min(max(a.len[(int64_t)b * a.beams + lane], 0), a.rows);
  }
  const bool moves = lane < a.beams && parent != lane;
  if (!__any(moves)) return;
  // the longest state that is read, and of each how many rows
  int most = __shfl(len, parent);
  most = moves ? most : 0;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) most = max(most, __shfl_xor(most, m));
  const int64_t units = (int64_t)most * a.cols;
  char* const state = a.state + (int64_t)blockIdx.z * a.layer_ld + (int64_t)b * a.beams * a.slot_ld;
  for (int64_t e0 = (int64_t)blockIdx.x * 256; e0 < units; e0 += (int64_t)gridDim.x * 256) {
    const int64_t e = e0 + threadIdx.x;
    const int row = (int)(e / a.cols), c = (int)(e - (int64_t)row * a.cols);
    char* const p = state + (int64_t)row * a.row_ld + (int64_t)c * sizeof(V);
    V x[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (j < a.beams && __any(moves && parent == j) && row < __builtin_amdgcn_readlane(len, j))
        x[j] = *reinterpret_cast<const V*>(p + j * a.slot_ld);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      uint64_t to = __ballot(moves && parent == j);
      if (to == 0) continue;
      const bool in = row < __builtin_amdgcn_readlane(len, j);
      while (to) {
        const int i = __builtin_ctzll(to);
        to &= to - 1;
        if (in) *reinterpret_cast<V*>(p + i * a.slot_ld) = x[j];
      }
    }
  }
}
}  // namespace

#define VRS_BEAM_PART(TN, T, VT)                                                                                              \
  extern "C" __global__ __launch_bounds__(256) void vrs_beam_part_##TN##_v##VT(vrs_beam_args a) { part_body<T, VT>(a); }
VRS_BEAM_PART(bf16, bf16_t, 1)
VRS_BEAM_PART(bf16, bf16_t, 4)
VRS_BEAM_PART(f32, float, 2)
VRS_BEAM_PART(f32, float, 8)
extern "C" __global__ __launch_bounds__(256) void vrs_beam_join_bf16(vrs_beam_args a) { join_body<bf16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_beam_join_f32(vrs_beam_args a) { join_body<float>(a); }
#define VRS_REORDER(VN, V)                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void vrs_beam_reorder_##VN##_n4(vrs_reorder_args a) { reorder_body<V, 4>(a); }  \
  extern "C" __global__ __launch_bounds__(256) void vrs_beam_reorder_##VN##_n8(vrs_reorder_args a) { reorder_body<V, 8>(a); }  \
  extern "C" __global__ __launch_bounds__(256) void vrs_beam_reorder_##VN##_n16(vrs_reorder_args a) { reorder_body<V, 16>(a); } \
  extern "C" __global__ __launch_bounds__(256) void vrs_beam_reorder_##VN##_n64(vrs_reorder_args a) { reorder_body<V, 64>(a); }
VRS_REORDER(b16, u32x4_t)
VRS_REORDER(b4, uint32_t)
VRS_REORDER(b1, uint8_t)
