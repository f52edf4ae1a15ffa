// Eviction from a cache, for gfx950: of a sequence's keys the first ones, the most
// recent ones and, up to the budget, those of the others that received the most
// attention stay, for each key head by itself and in their order.
//
// Two launches: the choice (a workgroup for each sequence and key head), then the
// move of K and V along the list of kept places.
#include "common.h"

namespace {

struct Keys {
  int64_t k0, o0;     // first row, and where the kept ones go
  int n;              // keys inside the buffer
};
__device__ __forceinline__ Keys keys_of(const vrs_evict_args& a, int i) {
  Keys s;
  s.k0 = a.k_start[i];
  s.o0 = a.o_start ? a.o_start[i] : s.k0;
  s.n = s.k0 < 0 || s.k0 >= a.k_rows ? 0 : (int)min((int64_t)max(a.k_len[i], 0), a.k_rows - s.k0);
  return s;
}

// Order of attention: as the numbers, both zeros alike, NaN above all.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// The choice.  The threshold is the largest T that at least m of the keys that
// compete reach, found two bits at a time by counting.
constexpr int kT = 1024, kHeld = 16;        // threads; keys of a thread in registers
__device__ __forceinline__ void choose_body(const vrs_evict_args& a) {
  __shared__ int cnt[2][3][kT / 64];
  __shared__ uint2 pre[2][kT / 64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = blockIdx.x % a.kv, seq = blockIdx.x / a.kv;
  const Keys s = keys_of(a, seq);
  const int n = s.n, keep = min(n, a.budget);
  int* kept = a.kept + ((int64_t)seq * a.kv + h) * a.budget;
  const float* acc = a.acc + s.k0 * a.acc_ld + h * a.acc_hd;
  float* acco = a.acco + s.o0 * a.acco_ld + h * a.acco_hd;
  const int last = max(n - a.recent, 0);                       // from here on all stay
  const int rounds = (n + kT - 1) / kT;
  const bool all = n <= a.budget;
  auto value = [&](int i) { return acc[(int64_t)i * a.acc_ld]; };
  uint32_t held[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int i = r * kT + tid;
    held[r] = !all && i >= a.first && i < last ? order_of(value(i)) : 0;   // (0: the order of no number)
  }
  const int m = keep - min(a.first, n) - (n - max(last, min(a.first, n)));    // of those that compete
  uint32_t T = 0;
  if (!all && m > 0) {
    for (int b = 30, turn = 0; b >= 0; b -= 2, turn ^= 1) {
      const uint32_t t1 = T | 1u << b, t2 = T | 2u << b, t3 = T | 3u << b;
      int c1 = 0, c2 = 0, c3 = 0;
      auto count = [&](uint32_t o) {
        c1 += __builtin_popcountll(__ballot(o >= t1));
        c2 += __builtin_popcountll(__ballot(o >= t2));
        c3 += __builtin_popcountll(__ballot(o >= t3));
      };
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
        if (r < rounds) count(held[r]);
      for (int r = kHeld; r < rounds; ++r) {
        const int i = r * kT + tid;
        count(i >= a.first && i < last ? order_of(value(i)) : 0);
      }
      if (lane == 0) cnt[turn][0][wave] = c1, cnt[turn][1][wave] = c2, cnt[turn][2][wave] = c3;
      __syncthreads();
      c1 = c2 = c3 = 0;
#pragma unroll
      for (int w = 0; w < kT / 64; ++w) c1 += cnt[turn][0][w], c2 += cnt[turn][1][w], c3 += cnt[turn][2][w];
      T = c3 >= m ? t3 : c2 >= m ? t2 : c1 >= m ? t1 : T;
    }
  }
  // how many equal ones stay: what the larger ones leave
  int above = 0;
  if (!all && m > 0) {
    int c = 0;
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
      if (r < rounds) c += __builtin_popcountll(__ballot(held[r] > T));
    for (int r = kHeld; r < rounds; ++r) {
      const int i = r * kT + tid;
      c += __builtin_popcountll(__ballot(i >= a.first && i < last && order_of(value(i)) > T));
    }
    __syncthreads();
    if (lane == 0) cnt[0][0][wave] = c;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) above += cnt[0][0][w];
  }
  const uint32_t equal = (uint32_t)max(m - above, 0);
  // places in order: those that stay anyway and those equal to T before each
  uint32_t sure0 = 0, eq0 = 0;
  for (int r = 0; r < rounds; ++r) {
    const int i = r * kT + tid;
    const float x = i < n ? value(i) : 0.f;
    const uint32_t o = order_of(x);
    const bool in = i < n, competes = in && i >= a.first && i < last;
    const bool sure = in && (all || !competes || (m > 0 && o > T)), eq = competes && !all && m > 0 && o == T;
    const uint64_t ms = __ballot(sure), me = __ballot(eq);
    if (lane == 0) pre[r & 1][wave] = make_uint2(__builtin_popcountll(ms), __builtin_popcountll(me));
    __syncthreads();                                           // also: the round's values are read
    uint32_t sb = sure0, eb = eq0;
#pragma unroll
    for (int w = 0; w < kT / 64; ++w) {
      const uint2 c = pre[r & 1][w];
      if (w < wave) sb += c.x, eb += c.y;
      sure0 += c.x, eq0 += c.y;
    }
    const uint64_t below = (1ull << lane) - 1;
    sb += __builtin_popcountll(ms & below);
    eb += __builtin_popcountll(me & below);
    if (sure || (eq && eb < equal)) {
      const uint32_t to = sb + min(eb, equal);
      if (to < (uint32_t)keep) {
        kept[to] = i;
        if (s.o0 >= 0 && s.o0 + to < a.o_rows) acco[(int64_t)to * a.acco_ld] = x;
      }
    }
  }
  for (int j = keep + tid; j < a.budget; j += kT) kept[j] = -1;
}

// The move: a workgroup takes a slice of the vectors of one head's rows, of K or of
// V, and passes over the kept places in order.  A kept key never moves up, so in
// place a tile's rows may be written once they are read: everything read later
// lies behind them.
template <typename V>
__device__ __forceinline__ void move_body(const vrs_evict_args& a) {
  constexpr int U = 8, NT = 256;
  const int tid = threadIdx.x;
  const int slice = blockIdx.x % a.slices, rest = blockIdx.x / a.slices, h = rest % a.kv, seq = rest / a.kv;
  const bool second = blockIdx.y == 1;
  const int64_t k0 = a.k_start[seq], o0 = a.o_start ? a.o_start[seq] : k0;
  const int* kept = a.kept + ((int64_t)seq * a.kv + h) * a.budget;
  const int c0 = (int)((int64_t)a.cols * slice / a.slices), c1 = (int)((int64_t)a.cols * (slice + 1) / a.slices), w = c1 - c0;
  // offsets are in vectors
  const int64_t ld = second ? a.v_ld : a.k_ld, hd = second ? a.v_hd : a.k_hd;
  const int64_t old_ = second ? a.vo_ld : a.ko_ld, ohd = second ? a.vo_hd : a.ko_hd;
  const V* src = static_cast<const V*>(second ? a.v : a.k) + k0 * ld + h * hd + c0;
  V* dst = static_cast<V*>(second ? a.vo : a.ko) + o0 * old_ + h * ohd + c0;
  const bool in_place = static_cast<const void*>(src) == static_cast<const void*>(dst);
  const int room = o0 < 0 || o0 >= a.o_rows ? 0 : (int)min((int64_t)a.budget, a.o_rows - o0);
  int total = 0;
  for (int64_t e0 = 0;; e0 += U * NT) {
    V x[U];
    int to[U];
    bool more = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = e0 + u * NT + tid;
      const int64_t row = e / w;
      const int c = (int)(e - row * w);
      const int from = row < a.budget ? kept[row] : -1;
      to[u] = -1;
      if (from >= 0) {
        more = true;
        if (row < room && !(in_place && from == row)) {
          x[u] = src[(int64_t)from * ld + c];
          to[u] = (int)row;
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!__syncthreads_or(more)) break;                        // the tile is read
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = e0 + u * NT + tid;
      if (to[u] >= 0) dst[(int64_t)to[u] * old_ + (e - e / w * w)] = x[u];
    }
  }
  if (!second && slice == 0 && h == 0 && a.len_out) {
    for (int j = tid; j < a.budget; j += NT) total += kept[j] >= 0;
    __shared__ int sum;
    if (tid == 0) sum = 0;
    __syncthreads();
    atomicAdd(&sum, total);
    __syncthreads();
    if (tid == 0) a.len_out[seq] = sum;
  }
}
}  // namespace

extern "C" __global__ __launch_bounds__(1024) void vrs_evict_choose(vrs_evict_args a) { choose_body(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b16(vrs_evict_args a) { move_body<u32x4_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b4(vrs_evict_args a) { move_body<uint32_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b2(vrs_evict_args a) { move_body<uint16_t>(a); }
