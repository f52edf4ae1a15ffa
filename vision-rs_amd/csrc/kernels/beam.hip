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
// is that of a vocabulary (k 16: some 40 of 8192).  Those that reach it go to LDS and
// each counts how many beat it, which is its place.  Where they are too many (equal
// or sorted logits) the workgroup takes its maximum k times instead.
//
// 32 requests of 8 beams over 128000 tokens in bfloat16, a quarter of them at their
// end (49 MB): 17 us for the chunks, 2.9 TB/s, and 10.2 for the join.  50 registers,
// so that 8 workgroups share a CU: with the next chunk's loads ahead it was 118 and
// 22 us.  A short chunk's elements one by one, all on their way at once, in place of
// its vectors: 77 and 18.4 us, for the whole chunks too.  Vector instructions take
// 45 % of the cycles (per logit: widening, maximum, FMA, v_exp at four times an
// instruction's cycles, addition, two comparisons), waits for the loads and two
// barriers the rest.
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

// A number that r lanes of the wave reach at least: the r-th largest order, its lower 16 bits cleared (0: none).
__device__ __forceinline__ uint32_t reached(uint32_t o, int r) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t trial = t | 1u << b;
    if (__builtin_popcountll(__ballot(o >= trial)) >= r) t = trial;
  }
  return t;
}

// Over the lanes of a wave by DPP: shifts inside rows of 16, then rows into the next; lane 63 has all.
template <int C, int ROWS>
__device__ __forceinline__ float dpp(float old, float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(x), C, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0x111, 0xf>(x, x));
  x = fmaxf(x, dpp<0x112, 0xf>(x, x));
  x = fmaxf(x, dpp<0x114, 0xf>(x, x));
  x = fmaxf(x, dpp<0x118, 0xf>(x, x));
  x = fmaxf(x, dpp<0x142, 0xa>(x, x));
  x = fmaxf(x, dpp<0x143, 0xc>(x, x));
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
template <int C, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)b, C, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(b >> 32), C, ROWS, 0xf, false);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// lane 63's is the sum
__device__ __forceinline__ double wave_sum(double x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  return dpp_add<0x143, 0xc>(x);
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
// A chunk of one row: VT vectors of 16 bytes to a thread.  The sum is of 2^(x L - R), L = log2 e rounded to float32
// and R = m L rounded, one FMA and one v_exp to a logit, and lse = (R + log2 sum) / L, so that R's rounding falls out
// and L's (1.3e-8) counts times the entropy only.  R is off by up to 2^-24 of itself, which the largest logit's term
// has in its exponent (a chunk masked by -1e10 would leave the range of 2^x): from |m| = 2^20 on the terms are
// 2^((x - m) L), of a difference that is exact where it counts, and R = m L in 64 bits.  A NaN or +infinity makes the
// sum NaN.
constexpr float kL = 1.44269502f;
constexpr float kNear = 1048576.f;
template <typename T, int VT>
__device__ __forceinline__ void part_body(const vrs_beam_args& a) {
  constexpr int V = 16 / (int)sizeof(T), N = VT * V;
  constexpr int kEach = kCand / kWaves;
  __shared__ __attribute__((aligned(16))) uint64_t cand[kWaves][kEach];
  __shared__ int count[kWaves];
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
  // Vectors of a row that starts anywhere.  A short chunk's go round the waves, so that each has its share; one of
  // fewer than k vectors is taken by elements, since each lane has but one number for the threshold (64 x 8 beams
  // over 849 tokens, k 128: 87 us by vectors, 40 by elements).
  constexpr int kThin = V * 128 / kT;          // elements of a thread at most (k <= 128)
  const bool whole = n == N * kT, thin = !whole && n < V * a.k;
  const int place = whole ? tid : lane * kWaves + wave;
  u32x4_t raw[VT];
  if (whole) {
#pragma unroll
    for (int j = 0; j < VT; ++j) __builtin_memcpy(&raw[j], x + (j * kT + place) * V, 16);
  } else {
    constexpr uint32_t kNo = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;                    // -infinity
#pragma unroll
    for (int j = 0; j < VT; ++j) {
      const int e0 = (j * kT + place) * V;
      raw[j] = (u32x4_t){kNo, kNo, kNo, kNo};
      if (thin) continue;
      if (e0 + V <= n) {
        __builtin_memcpy(&raw[j], x + e0, 16);
      } else if (e0 < n) {                     // the row ends in this vector
        T last[V];
        __builtin_memcpy(last, &raw[j], 16);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e0 + e < n) last[e] = x[e0 + e];
        __builtin_memcpy(&raw[j], last, 16);
      }
    }
    if (thin) {
      T own[V];
      __builtin_memcpy(own, &raw[0], 16);
#pragma unroll
      for (int e = 0; e < kThin; ++e)
        if (e * kT + tid < n) own[e] = x[e * kT + tid];
      __builtin_memcpy(&raw[0], own, 16);
    }
  }
  float v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(raw[i / 4][i % 4]);
    else v[i] = __uint_as_float(i % 2 ? raw[i / 8][i % 8 / 2] & 0xffff0000u : raw[i / 8][i % 8 / 2] << 16);
  }
  reinterpret_cast<u32x4_t*>(cand)[tid] = (u32x4_t){0, 0, 0, 0};    // the ranks below read whole eights
  reinterpret_cast<u32x4_t*>(cand)[kT + tid] = (u32x4_t){0, 0, 0, 0};
  const int token0 = c0 + (thin ? tid : place * V);
  auto token = [&](int i) { return (uint32_t)(token0 + (thin && i < kThin ? i * kT : (i / V) * kT * V + i % V)); };
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);                   // (a NaN is passed over)
  if (!(m > -INFINITY)) m = -INFINITY;                              // (nothing else but NaN)
  // what every wave has at least ceil(k / waves) numbers of
  const uint32_t top = m == -INFINITY ? 0 : order32(m);
  const uint32_t each = reached(top, (a.k + kWaves - 1) / kWaves);
  m = wave_max(m);
  if (lane == 0) swm[wave] = m, sth[wave] = each;
  __syncthreads();
  m = fmaxf(fmaxf(swm[0], swm[1]), fmaxf(swm[2], swm[3]));
  uint32_t T0 = min(min(sth[0], sth[1]), min(sth[2], sth[3]));
  if (T0 == 0 && a.k <= 64) {                  // some wave has not so many (masked tokens): one that has k, if any
    const uint32_t alone = reached(top, a.k);
    if (lane == 0) salone[wave] = alone;
    __syncthreads();
    T0 = max(max(salone[0], salone[1]), max(salone[2], salone[3]));
  }
  const float Tf = T0 ? __uint_as_float(T0 ^ ((int32_t)T0 < 0 ? 0x80000000u : 0xffffffffu)) : -3.40282347e38f;
  // candidates (none is -infinity or NaN), each wave's in its own part of the list
  int mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = v[i] >= Tf;
    const uint64_t mask = __ballot(in);
    if (mask == 0) continue;
    const int p = mine + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (in && p < kEach) cand[wave][p] = (uint64_t)order32(v[i]) << 32 | ~token(i);
    mine += __builtin_popcountll(mask);
  }
  if (lane == 0) count[wave] = mine;
  const float ref = m == -INFINITY ? 0.f : m;
  const bool near = fabsf(ref) < kNear;
  float sum = 0.f;
  if (near) {
    const float R = ref * kL;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[i], kL, -R));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) sum += __builtin_amdgcn_exp2f((v[i] - ref) * kL);
  }
  const double total = wave_sum(sum);
  if (lane == 63) sws[wave] = total;
  __syncthreads();
  const int64_t at = (int64_t)row * a.chunks + ch;
  if (tid == 0)
    a.part[at] = make_double2(near && m > -INFINITY ? (double)(ref * kL) : (double)m * kL, sws[0] + sws[1] + sws[2] + sws[3]);
  uint2* list = a.list + at * a.k;
  int have = 0, most = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) have += count[w], most = max(most, count[w]);
  auto logit = [](uint32_t o) { return o ^ (((int32_t)o >> 31) ? 0x80000000u : 0xffffffffu); };
  if (most <= kEach) {
    for (int i = lane; i < mine; i += 64) {
      const uint64_t me = cand[wave][i];       // larger logits, then smaller tokens, are larger numbers
      int rank = 0;
#pragma unroll 1
      for (int w = 0; w < kWaves; ++w) {
        const int n8 = count[w];
        for (int j = 0; j < n8; j += 8) {
#pragma unroll
          for (int e = 0; e < 8; ++e) rank += cand[w][j + e] > me;
        }
      }
      if (rank < a.k) list[rank] = make_uint2(logit((uint32_t)(me >> 32)), ~(uint32_t)me);
    }
    if (tid < a.k && tid >= have) list[tid] = make_uint2(0, 0xffffffffu);
  } else {
    uint64_t lo = ~0ull;
    uint32_t lat = 0;                          // the last one taken
    for (int k = 0; k < a.k; ++k) {
      uint64_t o = 0;
      uint32_t p = 0xffffffffu;
      for (int e = tid; e < n; e += kT) {      // (from memory again: rare, so small code rather than fast)
        const float f = Elt<T>::to_f(x[e]);
        const uint32_t q = (uint32_t)(c0 + e);
        const uint64_t c = f > -INFINITY ? order32(f) : 0;
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
  __shared__ __attribute__((aligned(16))) uint64_t co[kCand];
  __shared__ __attribute__((aligned(16))) uint32_t cat[kCand];
  __shared__ uint64_t ko[kCand];
  __shared__ uint32_t kat[kCand];
  __shared__ __attribute__((aligned(16))) uint32_t smax[kT];
  __shared__ int count, kept;
  __shared__ uint32_t sth;
  __shared__ uint64_t so[kWaves];
  __shared__ uint32_t sat[kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, b = blockIdx.x;
  // Lists are in order, so the first `per` entries of a list are its largest: a thread takes every per-th from
  // one of them, and the k-th largest of the threads' first ones is reached by k entries at least.
  const int lists = a.beams * a.chunks;
  int per = 1, lg = 0;
  while (per * 2 * lists <= kT) per *= 2, ++lg;
  const int l0 = tid >> lg, j0 = tid & (per - 1);
  const uint2* base = a.list + (int64_t)b * lists * a.k;
  // (loaded early; a beam at its end has no lists, and what lies there is not used)
  constexpr int kEarly = 4;
  uint2 early[kEarly];
#pragma unroll
  for (int i = 0; i < kEarly; ++i) {
    const int j = j0 + i * per;
    early[i] = l0 < lists && j < a.k ? base[(int64_t)l0 * a.k + j] : make_uint2(0, 0xffffffffu);
  }
  // lse of a beam: 2^w lanes over its chunks
  int w = 0;
  while ((1 << w) < a.chunks && w < 6) ++w;
  for (int i0 = 0; i0 < a.beams; i0 += kT >> w) {
    const int i = i0 + (tid >> w), c0 = tid & ((1 << w) - 1);
    const bool in = i < a.beams;
    const int64_t row = (int64_t)b * a.beams + i;
    const float s = in ? a.scores[row] : 0.f;
    double m = -INFINITY, l = 0;
    double2 p = make_double2(-INFINITY, 0);
    if (in && c0 < a.chunks) p = a.part[row * a.chunks + c0];
    const bool done = in && a.done && a.done[row], mine = in && !done;
    for (int c = c0; mine && c < a.chunks; c += 64) m = fmax(m, c == c0 ? p.x : a.part[row * a.chunks + c].x);
    for (int k = 1; k < 1 << w; k <<= 1) m = fmax(m, __shfl_xor(m, k));
    for (int c = c0; mine && c < a.chunks; c += 64) {
      if (c != c0) p = a.part[row * a.chunks + c];
      l += p.y == 0.0 ? 0.0 : p.y * exp2(p.x - m);       // (a NaN stays one)
    }
    for (int k = 1; k < 1 << w; k <<= 1) l += __shfl_xor(l, k);
    if (in && c0 == 0) {
      score[i] = s;
      lse[i] = (m + log2(l)) / (double)kL;
      kind[i] = !(s - s == 0.f) ? 0 : done ? 2 : !(l > 0.0 && l < INFINITY && m > -INFINITY && m < INFINITY) ? 0 : 1;
    }
  }
  if (tid == 0) count = 0, kept = 0, sth = 0;
  __syncthreads();
  const float inv_chunks = 1.f / (float)a.chunks;
  // an entry's order (0: none) and flat place
  auto valued = [&](int l, int j, uint2 e, uint64_t& o, uint32_t& at) {
    int c;
    const int i = fdivmod(l, a.chunks, inv_chunks, c), k = kind[i];
    o = 0;
    if (k == 1 && e.y != 0xffffffffu) {
      o = order64(score[i] + ((double)__uint_as_float(e.x) - lse[i]));
      at = (uint32_t)(i * a.vocab) + e.y;
    } else if (k == 2 && j == 0 && c == 0) {
      o = order64(score[i]);
      at = (uint32_t)(i * a.vocab + a.eos);
    }
  };
  auto entry = [&](int l, int j, uint64_t& o, uint32_t& at) {
    valued(l, j, base[(int64_t)l * a.k + j], o, at);
  };
  uint32_t top = 0;
  for (int l = l0; l < lists; l += kT >> lg) {
    uint64_t o = 0;
    uint32_t at = 0;
    if (l == l0) valued(l, j0, early[0], o, at);
    else if (j0 < a.k) entry(l, j0, o, at);
    top = max(top, (uint32_t)(o >> 32));
  }
  smax[tid] = top;
  __syncthreads();
  int above = 0, reach = 0;
#pragma unroll 8
  for (int j = 0; j < kT / 4; ++j) {
    const u32x4_t c = reinterpret_cast<const u32x4_t*>(smax)[j];
#pragma unroll
    for (int e = 0; e < 4; ++e) above += c[e] > top, reach += c[e] >= top;
  }
  if (above < a.k && reach >= a.k) sth = top;
  __syncthreads();
  uint32_t T0 = max(sth, 1u);
  // what reaches T0: a thread's entries eight at a time, on their way together
  auto collect = [&]() {
    auto take = [&](uint64_t o, uint32_t at) {
      if ((uint32_t)(o >> 32) < T0) return false;
      const int p = atomicAdd(&count, 1);
      if (p < kCand) co[p] = o, cat[p] = at;
      return true;
    };
    for (int l = l0; l < lists; l += kT >> lg) {
      bool more = true;
      int j = j0;
      if (l == l0) {
#pragma unroll
        for (int i = 0; i < kEarly; ++i, j += per) {
          uint64_t o = 0;
          uint32_t at = 0;
          if (more) valued(l0, j, early[i], o, at);
          more = more && take(o, at);
        }
      }
      for (; more && j < a.k; j += 8 * per) {
        uint2 e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = j + i * per < a.k ? base[(int64_t)l * a.k + j + i * per] : make_uint2(0, 0xffffffffu);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint64_t o = 0;
          uint32_t at = 0;
          if (more) valued(l, j + i * per, e[i], o, at);
          more = more && take(o, at);
        }
      }
    }
    __syncthreads();
    return count;
  };
  int have = collect();
  // The k-th largest (in the upper bits) of those that LDS holds bounds that of all.
  auto bound = [&]() {
    uint32_t mine[kCand / kT], t = 0;
#pragma unroll
    for (int i = 0; i < kCand / kT; ++i) mine[i] = i * kT + tid < have ? (uint32_t)(co[i * kT + tid] >> 32) : 0;
    for (int bit = 31; bit >= 6; --bit) {
      const uint32_t trial = t | 1u << bit;
      int c = 0;
#pragma unroll
      for (int i = 0; i < kCand / kT; ++i) c += __builtin_popcountll(__ballot(mine[i] >= trial));
      if (lane == 0) smax[(bit & 1) * kWaves + wave] = c;
      __syncthreads();
      const u32x4_t n = reinterpret_cast<const u32x4_t*>(smax)[bit & 1];
      if ((int)(n[0] + n[1] + n[2] + n[3]) >= a.k) t = trial;
    }
    return t;
  };
  if (have > kCand) {                          // beams of like scores
    const uint32_t T1 = bound();
    if (T1 > T0) {
      T0 = T1;
      __syncthreads();                         // the count is read
      if (tid == 0) count = 0;
      __syncthreads();
      have = collect();
    }
  }
  // Ranks cost their number squared: those that cannot be among the k leave first.
  uint64_t* ro = co;
  uint32_t* rat = cat;
  int ranked = min(have, kCand);
  if (have > 2 * a.k + 32 && have <= kCand) {
    const uint32_t T1 = bound();
    for (int i = tid; i < have; i += kT) {
      if ((uint32_t)(co[i] >> 32) < T1) continue;
      const int p = atomicAdd(&kept, 1);
      ko[p] = co[i], kat[p] = cat[i];
    }
    __syncthreads();
    ro = ko, rat = kat;
    ranked = kept;
  }
  auto put = [&](int k, uint64_t o, uint32_t at) {
    const uint64_t bits = o ^ (((int64_t)o >> 63) ? 0x8000000000000000ull : ~0ull);
    a.out_scores[(int64_t)b * a.k + k] = (float)__builtin_bit_cast(double, bits);
    a.out_parents[(int64_t)b * a.k + k] = (int32_t)(at / (uint32_t)a.vocab);
    a.out_tokens[(int64_t)b * a.k + k] = (int32_t)(at % (uint32_t)a.vocab);
  };
  int got = min(have, a.k);
  if (have <= kCand) {
    for (int i = tid; i < ranked; i += kT) {
      const uint64_t o = ro[i];
      const uint32_t at = rat[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < ranked; ++j) r += ro[j] > o || (ro[j] == o && rat[j] < at);
      if (r < a.k) put(r, o, at);
    }
  } else {
    uint64_t lo = ~0ull;
    uint32_t lat = 0;
    for (int k = 0; k < a.k; ++k) {
      uint64_t o = 0;
      uint32_t p = 0xffffffffu;
      for (int l = l0; l < lists; l += kT >> lg)
        for (int j = j0; j < a.k; j += per) {
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
// writes them to where they go; no other thread touches that vector.  16 requests of 8
// beams, 60 .. 300 rows of 4 KiB in 16 layers, 1.5 GB: 300 .. 321 us, 4.8 .. 5.1 TB/s.
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
