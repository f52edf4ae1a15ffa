// What a workgroup of the attention kernels does with one job: a row tile of one key
// head against a part of one run of keys.
#pragma once
#include "attention_wave.h"

namespace {
// Where a workgroup's rows and keys lie, and where its results go.
struct AttentionJob {
  SeqSpan sp;
  int hk;               // key head
  int tile, step;       // row tile (few rows: the first, and the distance to the next)
  int part, parts;      // which part of how many of the keys
  int out_part;         // which part of the workspace; direct: results go to `out`, finished
  int causal;
  bool direct;
  int part_len;         // keys of a part (the last one takes what is left); 0: parts of one length
  int joined;           // prompts: finished results take in so many parts of the workspace, of so many keys in all
  int joined_keys;
};
// Keys [kb, ke) of a job's part of `keys`.
__device__ __forceinline__ void keys_of(const AttentionJob& job, int keys, int unit, int& kb, int& ke) {
  if (job.part_len == 0) return part_of(keys, job.part, job.parts, unit, kb, ke);
  kb = (int)min((int64_t)job.part * job.part_len, (int64_t)keys);
  ke = job.part == job.parts - 1 ? keys : (int)min((int64_t)(job.part + 1) * job.part_len, (int64_t)keys);
}

// The prompts' K and V tiles; one object for all bodies of a kernel that name it.
template <typename T, int D, int KT>
__device__ __forceinline__ T* prompt_lds() {
  __shared__ __attribute__((aligned(16))) T smem[3 * 2 * KT * D];
  return smem;
}

// ---------------------------------------------------------------------------
// Prompts: a workgroup of 4 waves takes 128 * QT rows, the queries of all heads
// of one key head (neighbouring rows share a query, so causal tiles waste
// little and the keys serve the whole group), a wave 32 * QT of them; K and V
// tiles of KT keys are shared through LDS.
//
// The loop is written as a software pipeline: the next 32 keys' scores are
// multiplied between these 32 keys' maximum and their exponentials, so that
// neither kind of instruction waits for the other's results.  Measured per 32
// keys x 32 queries and SIMD: 512 cycles of matrix instructions and 459 of
// vector ones in 1020 at D = 128, 256 and 475 in 713 at D = 64: close to their
// sums, so the waves of a SIMD hardly overlap one kind with the other, and
// neither unit is full (50 and 45 % at 128, 36 and 67 % at 64).
//
// LDS holds three tiles, filled by loads that go straight there: one barrier
// before tile i's last 32 keys (whose step reads tile i + 1's first scores)
// makes tile i + 1 visible and frees tile i - 1's place for tile i + 2, whose
// loads then have a whole tile's time.  Tiles that some row does not see whole
// take the general form of the step; the others three at a time, so that LDS
// addresses are constants.
//
// 8192 causal queries, 32 heads on 8 of 128: 500 .. 540 us queued (cards and
// their clock under this load differ), 1020 .. 1100 TFLOP/s; an 8192^3 product
// reaches 1110 .. 1160.  Traced one by one: 568 us at 1.86 GHz, 1.05 M cycles,
// rising to 670 as the clock falls to 1.52.  No LDS bank conflicts.  8 waves and
// 64-key tiles against 4 waves and 32: 516 us to 548.  At head sizes up to 64 the
// same exponentials serve half the products: 24 images of 196 .. 1600 patches,
// 12 heads: 120 .. 128 us, 700 TFLOP/s; four 4-wave workgroups on a CU with
// 32-key tiles against three with 64: 124 us to 130; two query tiles to a wave
// for the large (4096 x 32 heads: 148 us to 159).  Heads of 72 .. 120 run padded
// to 128 (64 sequences of 512, 16 heads: 64 113 us, 72 177, 80 180, 96 191, 128
// 207).  float32 is bound by its matrix instructions (64 cycles each).
template <typename T, int D, int KT, int QT, int NW>
__device__ __forceinline__ void prompt_body(const vrs_attention_args& a, const AttentionJob& job) {
  constexpr int NT = 64 * NW, BM = 32 * NW * QT, NS = KT / 32;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = KT * CH / NT;                 // chunks a thread stages of K, and of V
  constexpr int TILE = KT * D;
  __shared__ int odd_tile[3];     // first key of the tile that a buffer holds, if it had values not finite
  const int tid = threadIdx.x, wave = tid >> 6;
  const int hk = job.hk;
  const int group = a.heads / a.kv;
  const SeqSpan sp = job.sp;
  const int64_t rows = (int64_t)sp.q_len * group;
  const int tiles = (int)((rows + BM - 1) / BM);
  if (job.tile >= tiles) return;
  const int64_t r0 = (int64_t)(tiles - 1 - job.tile) * BM;     // late rows (causal: the most keys) first

  const Log2 u(a.c);
  Wave<T, D, QT> w;
  w.init(u);
  int64_t qrow[QT];
  int head[QT];
  bool ok[QT];
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    const int64_t r = r0 + wave * 32 * QT + q * 32 + w.l32;
    ok[q] = r < rows;
    const int j = (int)(min(r, rows - 1) / group);
    head[q] = hk * group + (int)(min(r, rows - 1) - (int64_t)j * group);
    qrow[q] = sp.q0 + j;
    w.lim[q] = visible(sp, j, job.causal);
    w.load_q(q, static_cast<const T*>(a.q) + qrow[q] * a.q_ld + head[q] * a.q_hd, a.dim, ok[q]);
  }
  int kb, ke;
  keys_of(job, visible(sp, (int)((min(r0 + BM, rows) - 1) / group), job.causal), KT, kb, ke);
  const int all = visible(sp, (int)(r0 / group), job.causal);   // keys that every row of the workgroup sees
  const int mine = __builtin_amdgcn_readlane(w.lim[QT - 1], 31);   // keys that some row of the wave sees

  const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
  const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
  // A thread's chunks of a tile, straight to LDS: one instruction of a wave fills 1 KiB in lane
  // order, so the swizzle is in what each lane loads.  Elements past the head and keys past the
  // sequence's last are out of the buffer's range and fill in 0; such keys are masked besides.
  uint32_t ko[IT], vo[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int slot = (i * NW + wave) * 64 + (tid & 63), row = slot / CH, at = slot % CH;
    const int kc = (at ^ Lds<T, D>::kswz(row)) * PER, vc = (at ^ Lds<T, D>::vswz(row)) * PER;
    ko[i] = kc < a.dim ? (uint32_t)(row * (int)a.k_ld + kc) * (uint32_t)sizeof(T) : kOOB;
    vo[i] = vc < a.dim ? (uint32_t)(row * (int)a.v_ld + vc) * (uint32_t)sizeof(T) : kOOB;
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)prompt_lds<T, D, KT>() + wave * 1024);
  auto load = [&](int buf, int kc) {
    const int n = min(KT, sp.k_lim - kc);
    const i32x4_hw rk = lds_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
    const i32x4_hw rv = lds_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((n - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
    const uint32_t to = lds0 + buf * 2 * TILE * (uint32_t)sizeof(T);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_lds(rk, ko[i], to + i * NW * 1024);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_lds(rv, vo[i], to + TILE * (uint32_t)sizeof(T) + i * NW * 1024);
  };
  // V of a tile that some row does not see whole: values that are not finite become 0
  auto clean_tile = [&](int buf, int kc) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      u32x4_t* at = reinterpret_cast<u32x4_t*>(prompt_lds<T, D, KT>() + (buf * 2 + 1) * TILE) + (i * NW + wave) * 64 + (tid & 63);
      u32x4_t u = *at;
      if (clean<T>(u)) {
        *at = u;
        bad = true;
      }
    }
    if (bad) odd_tile[buf] = kc;
  };
  if (kb < ke) {
    if (tid < 3) odd_tile[tid] = -1;
    load(0, kb);
    if (kb + KT < ke) {
      load(1, kb + KT);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * IT) : "memory");   // the first tile is there
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
    f32x16_t s[QT];
    float t[QT];
    int kc = kb;
    // maximum of 32 keys' scores, of which those a query does not see are masked first
    auto look = [&](bool masked, int key) {
#pragma unroll
      for (int q = 0; q < QT; ++q) {
        if (masked) w.mask(q, s[q], key);
        t[q] = w.top(s[q]);
      }
    };
    w.scores(prompt_lds<T, D, KT>(), 0, s);
    look(kb + 32 > all, kb);
    // TAIL: some row does not see the whole of this or the next tile, or no tile follows
    auto tile = [&](auto tail, int buf, bool more) {
      constexpr bool TAIL = decltype(tail)::value;
      const int nbuf = buf == 2 ? 0 : buf + 1;
      const T* sK = prompt_lds<T, D, KT>() + buf * 2 * TILE;
      if (TAIL && kc + KT > all) clean_tile(buf, kc);
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const bool last = n == NS - 1;
        const bool live = !TAIL || kc + n * 32 < mine;
        if (live) w.follow(t, u);
        if (last) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the next tile
        if (last || (TAIL && kc + KT > all)) __syncthreads();
        if (last && kc + 2 * KT < ke) load(buf == 0 ? 2 : buf - 1, kc + 2 * KT);
        f32x16_t s1[QT];
        const bool ahead = !TAIL || ((!last || more) && kc + (n + 1) * 32 < mine);
        __builtin_amdgcn_s_setprio(1);
        if (ahead) w.scores(last ? prompt_lds<T, D, KT>() + nbuf * 2 * TILE : sK, last ? 0 : (n + 1) * 32, s1);
        if (live) {
          typename Wave<T, D, QT>::P p[QT];
#pragma unroll
          for (int q = 0; q < QT; ++q) p[q] = w.probs(q, s[q], u);
          w.pv(sK + TILE, n * 32, p);
        }
        __builtin_amdgcn_s_setprio(0);
        if (ahead) {
#pragma unroll
          for (int q = 0; q < QT; ++q) s[q] = s1[q];
          look(TAIL && kc + (n + 2) * 32 > all, kc + (n + 1) * 32);
        }
      }
      if (TAIL && odd_tile[buf] == kc)
        for (int n = 0; n < NS; ++n)
          w.add_specials(vp + (int64_t)(kc + n * 32) * a.v_ld, a.v_ld, sp.k_lim - kc - n * 32, a.dim, kc + n * 32);
      kc += KT;
    };
    while (kc + 4 * KT <= all && kc + 3 * KT < ke) {     // three at a time: LDS addresses are constants
      tile(std::false_type{}, 0, true);
      tile(std::false_type{}, 1, true);
      tile(std::false_type{}, 2, true);
    }
    for (int buf = 0; kc < ke; buf = buf == 2 ? 0 : buf + 1) tile(std::true_type{}, buf, kc + KT < ke);
  }
  if (job.joined) {
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      const int64_t i = qrow[q] * a.heads + head[q];
      w.take_parts(q, a.part_o + i * a.dim, a.part_rl + i, (int64_t)a.s.q_rows * a.heads, job.joined, a.dim, u);
      w.lim[q] = (int)min((int64_t)w.lim[q] + job.joined_keys, (int64_t)0x7fffffff);
    }
  }
#pragma unroll
  for (int q = 0; q < QT; ++q) {
    if (job.direct) {
      w.store(q, static_cast<T*>(a.out) + qrow[q] * a.o_ld + head[q] * a.o_hd, a.dim, ok[q]);
    } else {
      const int64_t i = ((int64_t)job.out_part * a.s.q_rows + qrow[q]) * a.heads + head[q];
      w.store_part(q, a.part_o + i * a.dim, a.part_rl + i, a.dim, ok[q]);
    }
  }
}

// ---------------------------------------------------------------------------
// Few queries to a sequence (single tokens): a workgroup takes 32 rows, the
// queries of all heads of one key head, so that the keys are read once for
// the group; its NW waves take different tiles of 32 keys, each on its own (no
// barrier inside the loop), and join their O, m and l through LDS at the end.
// Memory bound: K goes straight to registers in operand layout (16 bytes of a
// row to a lane), V through a wave's own LDS tile for the transposed reads,
// the next tile's loads in flight meanwhile.  64 tokens over 500 .. 8000 keys,
// 32 heads on 8 of 128, 1.14 GB: 233 us, 4.9 TB/s.
// SHARED: in the LDS of the prompts' body, for a kernel that has both.  It holds the
// O of two waves, so that the upper two are added to the lower two first.
template <typename T, int D, int NW, bool SHARED = false>
__device__ __forceinline__ void few_body(const vrs_attention_args& a, const AttentionJob& job) {
  using E = Elt<T>;
  using G = typename E::group;
  constexpr int CH = Lds<T, D>::CH, PER = 16 / (int)sizeof(T);
  constexpr int IT = 32 * CH / 64;                 // V chunks of a lane
  constexpr int OL = D + 4;                        // O row in LDS (float32)
  constexpr int V_BYTES = NW * 32 * D * (int)sizeof(T), O_BYTES = NW * 32 * OL * 4;
  static_assert(!SHARED || (NW == 4 && (V_BYTES > O_BYTES / 2 ? V_BYTES : O_BYTES / 2) <= 6 * 32 * D * (int)sizeof(T)), "");
  __shared__ __attribute__((aligned(16))) char mem[SHARED ? 16 : V_BYTES > O_BYTES ? V_BYTES : O_BYTES];
  __shared__ float sR[NW][32], sl[NW][32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int hk = job.hk;
  const SeqSpan sp = job.sp;
  const int G_ = a.heads / a.kv;
  const int64_t rows = (int64_t)sp.q_len * G_;
  T* sV;
  float* sO;
  if constexpr (SHARED) {
    sV = prompt_lds<T, D, 32>() + wave * 32 * D;
    sO = reinterpret_cast<float*>(prompt_lds<T, D, 32>());
  } else {
    sV = reinterpret_cast<T*>(mem) + wave * 32 * D;
    sO = reinterpret_cast<float*>(mem);
  }

  const Log2 u(a.c);
  // row tiles of the sequence, one workgroup each (and more than were counted on, in turn)
  for (int64_t r0 = (int64_t)job.tile * 32; r0 < rows; r0 += (int64_t)job.step * 32) {
    Wave<T, D, 1> w;
    w.init(u);
    const int64_t pr = min(r0 + w.l32, rows - 1);
    const bool ok = r0 + w.l32 < rows;
    const int j = (int)(pr / G_), h = hk * G_ + (int)(pr - (int64_t)j * G_);
    const int64_t row = sp.q0 + j;
    const int lim = visible(sp, j, job.causal);
    w.lim[0] = lim;
    w.load_q(0, static_cast<const T*>(a.q) + row * a.q_ld + h * a.q_hd, a.dim, ok);
    const int lim_min = __builtin_amdgcn_readfirstlane(lim), lim_max = __builtin_amdgcn_readlane(lim, 31);
    int kb, ke;
    keys_of(job, lim_max, 32, kb, ke);

    const T* kp = static_cast<const T*>(a.k) + sp.k0 * a.k_ld + (int64_t)hk * a.k_hd;
    const T* vp = static_cast<const T*>(a.v) + sp.k0 * a.v_ld + (int64_t)hk * a.v_hd;
    G kr[D / 16];
    u32x4_t vr[IT];
    uint32_t ko[D / 16], vo[IT];           // offsets in a tile; elements past the head read 0
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const int d = i * 16 + w.hh * 8;
      ko[i] = d < a.dim ? (uint32_t)(w.l32 * (int)a.k_ld + d) * (uint32_t)sizeof(T) : kOOB;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int it = lane + i * 64, r = it / CH, ch = it % CH;
      vo[i] = ch * PER < a.dim ? (uint32_t)(r * (int)a.v_ld + ch * PER) * (uint32_t)sizeof(T) : kOOB;
    }
    auto load = [&](int kc) {              // keys past the sequence's last are masked, whatever they read
      const int n = min(32, sp.k_lim - kc);
      const auto rk = make_rsrc(kp + (int64_t)kc * a.k_ld, (int)(((n - 1) * a.k_ld + a.dim) * (int)sizeof(T)));
      const auto rv = make_rsrc(vp + (int64_t)kc * a.v_ld, (int)(((n - 1) * a.v_ld + a.dim) * (int)sizeof(T)));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) kr[i] = E::bload(rk, ko[i], 0);
#pragma unroll
      for (int i = 0; i < IT; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, vo[i], 0, 0);
    };
    int kc = kb + wave * 32;
    if (kc < ke) load(kc);
    while (kc < ke) {
      f32x16_t s[1];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) s[0] = mfma32_k16(kr[i], w.qf[0][i], s[0]);
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
      kc += NW * 32;
      if (kc < ke) load(kc);
      if (masked) w.mask(0, s[0], at);
      const float t[1] = {w.top(s[0])};
      w.follow(t, u);
      const typename Wave<T, D, 1>::P p[1] = {w.probs(0, s[0], u)};
      w.pv(sV, 0, p);
      if (__any(bad)) w.add_specials(vp + (int64_t)at * a.v_ld, a.v_ld, sp.k_lim - at, a.dim, at);
      __builtin_amdgcn_wave_barrier();
    }
    // join the waves: the largest reference, sums and O scaled to it
    float lt = sum32(w.l[0]);
    constexpr int NJ = SHARED ? 2 : NW;    // of so many waves
    auto put = [&](int at) {
      if (w.hh == 0) {
        sR[at][w.l32] = w.R[0];
        sl[at][w.l32] = lt;
      }
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4_t*>(&sO[(at * 32 + w.l32) * OL + d * 32 + g * 8 + w.hh * 4]) =
              (f32x4_t){w.o[0][d][4 * g], w.o[0][d][4 * g + 1], w.o[0][d][4 * g + 2], w.o[0][d][4 * g + 3]};
    };
    __syncthreads();                       // every wave is done with its V tile
    if constexpr (SHARED) {
      if (wave >= 2) put(wave - 2);
      __syncthreads();
      if (wave < 2) {
        const float other = sR[wave][w.l32], mx = fmaxf(w.R[0], other);
        const float mine = u.factor(w.R[0], mx), its = u.factor(other, mx);
        lt = mine * lt + its * sl[wave][w.l32];
        w.R[0] = mx;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&sO[(wave * 32 + w.l32) * OL + d * 32 + g * 8 + w.hh * 4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) w.o[0][d][4 * g + k] = mine * w.o[0][d][4 * g + k] + its * v[k];
          }
        put(wave);                         // where it has read, and no other wave has
      }
    } else {
      put(wave);
    }
    __syncthreads();
    // 2 NW threads to a row, 4 elements at a time
    const int rr = threadIdx.x / (2 * NW), e0 = threadIdx.x % (2 * NW) * 4;
    if (r0 + rr < rows) {
      const int jj = (int)((r0 + rr) / G_), ho = hk * G_ + (int)(r0 + rr - (int64_t)jj * G_);
      const int64_t orow = sp.q0 + jj;
      float mx = sR[0][rr];
#pragma unroll
      for (int i = 1; i < NJ; ++i) mx = fmaxf(mx, sR[i][rr]);
      float f[NJ], lsum = 0.f;
#pragma unroll
      for (int i = 0; i < NJ; ++i) {       // a wave without keys has l = 0, O = 0
        f[i] = u.factor(sR[i][rr], mx);
        lsum += f[i] * sl[i][rr];
      }
      const float inv = job.direct ? share(lsum, visible(sp, jj, job.causal)) : 1.f;
      const int64_t at = ((int64_t)job.out_part * a.s.q_rows + orow) * a.heads + ho;
      if (!job.direct && e0 == 0) a.part_rl[at] = make_float2(mx, lsum);
      T* out = static_cast<T*>(a.out) + orow * a.o_ld + ho * a.o_hd;
      for (int e = e0; e < a.dim; e += 8 * NW) {
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NJ; ++i) v += f[i] * *reinterpret_cast<const f32x4_t*>(&sO[(i * 32 + rr) * OL + e]);
        v *= inv;
        if (!job.direct) {
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

}  // namespace
