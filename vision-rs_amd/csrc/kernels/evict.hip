// Eviction from a cache, for gfx950: of a sequence's keys the first ones, the most
// recent ones and, up to the budget, those of the others that received the most
// attention stay, for each key head by itself and in their order.
//
// Two launches: the choice (a workgroup for each sequence and key head), then the
// move of K and V along the list of kept places.  16 caches of 2500 .. 8000 keys, 8
// heads of 128 in bfloat16, cut to 2048 where they lie (274 MB): 23 us, bound by the
// rounds of counting in 128 workgroups, and 54, 4.9 TB/s (75 without the next tile's
// rows on their way; slices of 64 bytes of a row, half a cache line, 90).
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

// Sum over W lanes of a row of 16 whose lanes repeat after W, and over the lanes up to each of the first W.
template <int W>
__device__ __forceinline__ int row_sum(int x) {
  if constexpr (W == 16) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);    // row_ror 8, 4, 2, 1
    x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, true);
  }
  x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, true);
  return x + __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, true);
}
template <int W>
__device__ __forceinline__ int row_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);      // row_shr 1, 2, 4, 8: 0 comes in
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  if constexpr (W == 16) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  }
  return x;
}

// The choice.  The threshold is the largest T that at least m of the keys that
// compete reach, found two bits at a time by counting (a wave counts 64 keys with
// a comparison and a scalar popcount, and lane i of each wave reads wave i's
// counts), until one is reached by m keys and no more.
constexpr int kHeld = 16;                                // keys of a thread in registers
constexpr int kAtOnce = 4;                               // rounds of keys that are placed together
template <int kT>                                        // threads: 256 or 1024
__device__ __forceinline__ void choose_body(const vrs_evict_args& a) {
  constexpr int kW = kT / 64;
  __shared__ __attribute__((aligned(16))) int cnt[2][kW][4];
  __shared__ int2 pre[2][kAtOnce][kW];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int h = blockIdx.x % a.kv, seq = blockIdx.x / a.kv;
  const Keys s = keys_of(a, seq);
  const int n = s.n, keep = min(n, a.budget);
  int* kept = a.kept + ((int64_t)seq * a.kv + h) * a.budget;
  const float* acc = a.acc + s.k0 * a.acc_ld + h * a.acc_hd;
  float* acco = a.acco + s.o0 * a.acco_ld + h * a.acco_hd;
  const int first = min(a.first, n), last = max(n - a.recent, first);     // those between compete
  const int rounds = (n + kT - 1) / kT;
  const bool all = n <= a.budget;
  auto value = [&](int i) { return acc[(int64_t)i * a.acc_ld]; };
  float next[kAtOnce];
#pragma unroll
  for (int r = 0; r < kAtOnce; ++r) next[r] = r * kT + tid < n ? value(r * kT + tid) : 0.f;
  const int m = all ? 0 : keep - first - (n - last);           // of those that compete
  uint32_t T = 0;
  int above = 0;                                               // keys above T
  bool sharp = m == 0;                                         // those above T are m
  if (m == 0) T = 0xffffffffu;
  if (m > 0) {
    uint32_t held[kHeld];
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int i = r * kT + tid;
      held[r] = i >= first && i < last ? order_of(value(i)) : 0;          // (0: the order of no number)
    }
    int turn = 0;
    auto total = [&](int c1, int c2, int c3, int (&c)[3]) {
      if (lane == 0) *reinterpret_cast<int4*>(cnt[turn][wave]) = make_int4(c1, c2, c3, 0);
      __syncthreads();
      const int4 w = *reinterpret_cast<const int4*>(cnt[turn][lane & (kW - 1)]);
      c[0] = __builtin_amdgcn_readfirstlane(row_sum<kW>(w.x));
      c[1] = __builtin_amdgcn_readfirstlane(row_sum<kW>(w.y));
      c[2] = __builtin_amdgcn_readfirstlane(row_sum<kW>(w.z));
      turn ^= 1;
    };
    int c[3];
    for (int b = 30; b >= 0 && !sharp; b -= 2) {
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
        count(i >= first && i < last ? order_of(value(i)) : 0);
      }
      total(c1, c2, c3, c);
      const int reach = c[2] >= m ? c[2] : c[1] >= m ? c[1] : c[0];
      T = c[2] >= m ? t3 : c[1] >= m ? t2 : c[0] >= m ? t1 : T;
      sharp = reach == m;
    }
    if (sharp) {
      --T;                                                     // what is above that is what reaches T
    } else {
      int c1 = 0;
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
        if (r < rounds) c1 += __builtin_popcountll(__ballot(held[r] > T));
      for (int r = kHeld; r < rounds; ++r) {
        const int i = r * kT + tid;
        c1 += __builtin_popcountll(__ballot(i >= first && i < last && order_of(value(i)) > T));
      }
      total(c1, 0, 0, c);
      above = c[0];
    }
  }
  const int equal = sharp ? 0 : m - above;                     // the earliest of those equal to T stay too
  // places in order: those that stay anyway and those equal to T before each, kAtOnce rounds to a barrier
  int sure0 = 0, eq0 = 0;
  for (int r0 = 0, turn = 0; r0 < rounds; r0 += kAtOnce, turn ^= 1) {
    float x[kAtOnce];
    uint64_t ms[kAtOnce], me[kAtOnce];
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) x[r] = next[r];
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) {
      const int i = (r0 + kAtOnce + r) * kT + tid;
      if (i < n) next[r] = value(i);                           // (lies behind all that is written before)
    }
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) {
      const int i = (r0 + r) * kT + tid;
      const uint32_t o = order_of(x[r]);
      const bool competes = i >= first && i < last;
      ms[r] = __ballot(i < n && (all || !competes || o > T));
      me[r] = __ballot(competes && equal > 0 && o == T);
      if (lane == 0) pre[turn][r][wave] = make_int2(__builtin_popcountll(ms[r]), __builtin_popcountll(me[r]));
      asm volatile("" ::"v"(x[r]));
    }
    __syncthreads();                                           // also: the rounds' values are read
    const int2 c = pre[turn][lane >> 4][lane & (kW - 1)];      // a row of 16 lanes for each round
    const int ss = row_scan<kW>(c.x), es = row_scan<kW>(c.y);  // up to each wave
    const uint64_t bit = 1ull << lane;
#pragma unroll
    for (int r = 0; r < kAtOnce; ++r) {
      const int sb = sure0 + __builtin_amdgcn_readlane(ss, 16 * r + wave) - __builtin_popcountll(ms[r]) + __builtin_popcountll(ms[r] & (bit - 1));
      const int eb = eq0 + __builtin_amdgcn_readlane(es, 16 * r + wave) - __builtin_popcountll(me[r]) + __builtin_popcountll(me[r] & (bit - 1));
      sure0 += __builtin_amdgcn_readlane(ss, 16 * r + kW - 1);
      eq0 += __builtin_amdgcn_readlane(es, 16 * r + kW - 1);
      if ((ms[r] & bit) || ((me[r] & bit) && eb < equal)) {
        const int to = sb + min(eb, equal);
        if (to < keep) {
          kept[to] = (r0 + r) * kT + tid;
          if (s.o0 >= 0 && s.o0 + to < a.o_rows) acco[(int64_t)to * a.acco_ld] = x[r];
        }
      }
    }
  }
  for (int j = keep + tid; j < a.budget; j += kT) kept[j] = -1;
}

// The move: a workgroup takes a slice of the vectors of one head's rows, of K or of
// V, and passes over the kept places in order (where neither is moved in place,
// over a block of them).  A kept key never moves up, so in place a tile's rows may
// be written once they are read: everything read later lies behind them, and may
// be on its way already.
template <typename V>
__device__ __forceinline__ void move_body(const vrs_evict_args& a) {
  constexpr int U = 8, NT = 256;
  const int tid = threadIdx.x;
  const int slice = blockIdx.x % a.slices, rest = blockIdx.x / a.slices, h = rest % a.kv, seq = rest / a.kv;
  const bool second = blockIdx.y == 1;
  const int64_t k0 = a.k_start[seq], o0 = a.o_start ? a.o_start[seq] : k0;
  const int* kept = a.kept + ((int64_t)seq * a.kv + h) * a.budget;
  const int c0 = (int)((int64_t)a.cols * slice / a.slices), w = (int)((int64_t)a.cols * (slice + 1) / a.slices) - c0;
  // offsets are in vectors
  const int64_t ld = second ? a.v_ld : a.k_ld, hd = second ? a.v_hd : a.k_hd;
  const int64_t old_ = second ? a.vo_ld : a.ko_ld, ohd = second ? a.vo_hd : a.ko_hd;
  const V* const src = static_cast<const V*>(second ? a.v : a.k) + k0 * ld + h * hd + c0;
  V* const dst = static_cast<V*>(second ? a.vo : a.ko) + o0 * old_ + h * ohd + c0;
  const bool in_place = static_cast<const void*>(src) == static_cast<const void*>(dst);
  const int room = o0 < 0 || o0 >= a.o_rows ? 0 : (int)min((int64_t)a.budget, a.o_rows - o0);
  // w threads to a row (w <= NT), NT / w rows at a time
  const int rpp = NT / w, tr = tid / w, tc = tid - tr * w;
  const int b0 = (int)((int64_t)a.budget * blockIdx.z / gridDim.z), b1 = (int)((int64_t)a.budget * (blockIdx.z + 1) / gridDim.z);
  struct Tile { V x[U]; int from[U]; };      // from: the kept places, then those of them that move
  auto places = [&](Tile& t, int r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = r0 + u * rpp + tr;
      t.from[u] = tr < rpp && row < b1 ? kept[row] : -1;
    }
  };
  auto load = [&](Tile& t, int r0) {         // whether the tile has kept places
    bool any = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = r0 + u * rpp + tr;
      any |= t.from[u] >= 0;
      if (row >= room || (in_place && t.from[u] == row)) t.from[u] = -1;       // no room, or there already
      if (t.from[u] >= 0) t.x[u] = src[(int64_t)t.from[u] * ld + tc];
    }
    return any;
  };
  // one tile is loaded, the places of the next are known
  Tile t, n;
  places(t, b0);
  places(n, b0 + U * rpp);
  bool any = load(t, b0);
  for (int r0 = b0; r0 < b1; r0 += U * rpp) {
    const bool more = load(n, r0 + U * rpp);
    Tile n2;
    places(n2, r0 + 2 * U * rpp);
#pragma unroll
    for (int u = 0; u < U; ++u) asm volatile("" ::"v"(t.x[u]));
    if (!__syncthreads_or(any)) break;       // the tile is read
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t.from[u] >= 0) dst[(int64_t)(r0 + u * rpp + tr) * old_ + tc] = t.x[u];
    t = n;
    n = n2;
    any = more;
  }
  if (!second && slice == 0 && h == 0 && blockIdx.z == 0 && a.len_out && tid < 64) {
    int lo = 0, len = a.budget;                                            // the kept ones come first
    while (len > 1) {
      const int step = (len + 63) >> 6, i = tid * step;
      const uint64_t is = __ballot(i < len && kept[lo + i] >= 0);
      const int hit = is ? 63 - __builtin_clzll(is) : 0;
      lo += hit * step;
      len = min(step, len - hit * step);
    }
    if (tid == 0) a.len_out[seq] = lo + (kept[lo] >= 0);
  }
}
}  // namespace

extern "C" __global__ __launch_bounds__(256) void vrs_evict_choose_t256(vrs_evict_args a) { choose_body<256>(a); }
extern "C" __global__ __launch_bounds__(1024) void vrs_evict_choose_t1024(vrs_evict_args a) { choose_body<1024>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b16(vrs_evict_args a) { move_body<u32x4_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b4(vrs_evict_args a) { move_body<uint32_t>(a); }
extern "C" __global__ __launch_bounds__(256) void vrs_evict_move_b2(vrs_evict_args a) { move_body<uint16_t>(a); }
