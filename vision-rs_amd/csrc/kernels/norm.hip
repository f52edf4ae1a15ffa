// RMS norm of rows with the residual's addition, for gfx950.
//
//   s = x + res,  y = s * rsqrt(mean(s^2) + eps) * weight
//
// in float32 from the loads to the one rounding of each output (bfloat16,
// float32, or e4m3 on a fixed step, a step per row or per group of columns).
//
// Memory bound: x, res read once, sum, y written once.  TPR threads hold one
// row in registers between its two passes (sum of squares, then scaling), so
// a row is read once; a workgroup walks rows with the weights it needs in
// registers and the next row's loads in flight, which no branch holds up.
// 8192 rows of 4096 columns in bfloat16 with the residual, 268 MB: 43 us in
// bursts and 50 sustained, 6.2 and 5.3 TB/s (58 us without the loads ahead; a
// copy of 1 GiB moves 5.15 TB/s).
// Rows too wide for that (over 1024 vectors) lie in LDS as float32 between
// the passes, 1024 threads to a row.
#include "common.h"

namespace {
constexpr int kSame = 0, kFp8 = 1;
constexpr float kE4m3Max = 448.f;
constexpr float kMinNormal = 1.17549435e-38f;     // 2^-126

// VEC elements as they lie in memory (16 bytes, or one element), and as floats.
template <typename T, int VEC>
struct Raw {
  static_assert(VEC * sizeof(T) == 16, "one 16-byte load");
  u32x4_t u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const u32x4_t*>(p); }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[e]);
    else return __uint_as_float((e & 1) ? u[e / 2] & 0xffff0000u : u[e / 2] << 16);
  }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ float operator[](int) const { return Elt<T>::to_f(v); }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = Elt<T>::from_f(v[0]);
  } else {
    u32x4_t u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(v[i]);
      else u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
    *reinterpret_cast<u32x4_t*>(p) = u;
  }
}

// rne(clamp(v)) to e4m3; a NaN stays one (the clamp's minimum and maximum would drop it)
__device__ __forceinline__ float sat(float v) {
  return v != v ? v : __builtin_amdgcn_fmed3f(v, -kE4m3Max, kE4m3Max);
}
template <int VEC>
__device__ __forceinline__ void store_fp8(uint8_t* p, const float (&v)[VEC]) {
  static_assert(VEC % 4 == 0, "whole dwords");
  uint32_t u[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(v[4 * i]), sat(v[4 * i + 1]), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(v[4 * i + 2]), sat(v[4 * i + 3]), w, true);
    u[i] = (uint32_t)w;
  }
  if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(p) = u[0];
  else *reinterpret_cast<u32x2_t*>(p) = (u32x2_t){u[0], u[1]};
}

// Sum (or maximum) of one value per thread over the TPR threads of a row, on
// all of them; the order is fixed.
template <typename V, int TPR, bool MAX>
__device__ __forceinline__ V row_reduce(V v, V* lds) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const V o = __shfl_xor(v, m);
    if constexpr (MAX) v = v > o ? v : o;
    else v += o;
  }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    __syncthreads();                      // the array's earlier readers are done
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      if constexpr (MAX) v = v > lds[w] ? v : lds[w];
      else v += lds[w];
    }
  }
  return v;
}

// Whether a float32 sum of squares stands for its terms: neither they nor it left the type's range.
__device__ __forceinline__ bool in_range(float ss) { return ss > 1e-25f && ss < INFINITY; }

// How a maximum m of |y| scales to e4m3: by m / 448, by 1 where that is 0 (no values, or none that a
// scale could stand for).  Quotients by the scale are products with 448 / m as long as the scale is a
// normal number and so that inverse finite; by smaller scales (inv 0) they are divided.
struct Scale {
  float scale, inv;
  static __device__ __forceinline__ Scale step(float inv) { return {1.f, inv}; }
  static __device__ __forceinline__ Scale of(float m) {
    const float s = m / kE4m3Max;
    return {s > 0.f ? s : 1.f, m >= kE4m3Max * kMinNormal ? kE4m3Max / m : 0.f};
  }
};

// VEC elements of a row to e4m3, on `sc` or on the scale of their group, whose lanes are
// neighbours in a wave (all of them here, `in` or not).
template <int VEC>
__device__ __forceinline__ void put_fp8(const vrs_rms_args& a, int64_t row, int c, bool in, bool per_row, Scale sc,
                                        const float (&y)[VEC]) {
  if (a.group && !per_row) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) m = fmaxf(m, fabsf(y[e]));
    const int lanes = a.group / VEC;
    for (int d = 1; d < lanes; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    sc = Scale::of(m);
    if (in && c % a.group == 0) a.scales[row * (a.cols / a.group) + c / a.group] = sc.scale;
  }
  if (in) {
    float q[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) q[e] = y[e] * sc.inv;
    if (sc.inv == 0.f)
#pragma unroll
      for (int e = 0; e < VEC; ++e) q[e] = y[e] / sc.scale;
    store_fp8<VEC>(static_cast<uint8_t*>(a.y) + row * a.y_ld + c, q);
  }
}

template <typename T, int OUT, int TPR, int NV, int VEC>
__device__ __forceinline__ void rms_body(const vrs_rms_args& a) {
  constexpr int WG = 256, RPW = WG / TPR;      // rows of a workgroup's step
  __shared__ double lds_d[WG / 64];
  float* lds = reinterpret_cast<float*>(lds_d);
  const int t = threadIdx.x % TPR;
  const int sub = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);   // a row's threads are whole waves
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.res);
  T* sum = static_cast<T*>(a.sum);

  // Columns past the row's end load its last ones, and rows past the last that one again, so that no
  // load sits behind a branch; what they hold is dropped.
  int col[NV];
  float w[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = min((i * TPR + t) * VEC, a.cols - VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[i][e] = a.weight[col[i] + e];
  }
  Raw<T, VEC> nx[NV], nr[NV];
  auto fetch = [&](int64_t r0) {
    const int64_t row = min(r0 + sub, (int64_t)a.rows - 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) nx[i].load(x + row * a.x_ld + col[i]);
    if (res) {
#pragma unroll
      for (int i = 0; i < NV; ++i) nr[i].load(res + row * a.res_ld + col[i]);
    }
  };
  fetch((int64_t)blockIdx.x * RPW);
  // every thread of a workgroup makes every step (the reductions of wide rows have barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < a.rows; r0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = r0 + sub;
    const bool ok = row < a.rows;
    float s[NV][VEC];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      const bool in = ok && c < a.cols;
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] = !in ? 0.f : res ? nx[i][e] + nr[i][e] : nx[i][e];
      if (in && sum) store_vec<T, VEC>(sum + row * a.sum_ld + c, s[i]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += s[i][e] * s[i][e];
    }
    if (r0 + (int64_t)gridDim.x * RPW < a.rows) fetch(r0 + (int64_t)gridDim.x * RPW);
    ss = row_reduce<float, TPR, false>(ss, lds);
    float r;
    if (in_range(ss)) {
      r = 1.f / sqrtf(ss / (float)a.cols + a.eps);
    } else {     // the same sum in 64 bits
      double sd = 0.0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sd += (double)s[i][e] * (double)s[i][e];
      sd = row_reduce<double, TPR, false>(sd, lds_d);
      r = (float)(1.0 / sqrt(sd / (double)a.cols + (double)a.eps));
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[i][e] = s[i][e] * r * w[i][e];
        if constexpr (OUT == kFp8) amax = fmaxf(amax, fabsf(s[i][e]));
      }
    if constexpr (OUT == kSame) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (ok && c < a.cols) store_vec<T, VEC>(static_cast<T*>(a.y) + row * a.y_ld + c, s[i]);
      }
    } else {
      Scale sc = Scale::step(a.inv_step);
      const bool per_row = a.group == a.cols;
      if (per_row) {
        sc = Scale::of(row_reduce<float, TPR, true>(amax, lds));
        if (ok && t == 0) a.scales[row] = sc.scale;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        put_fp8<VEC>(a, row, c, ok && c < a.cols, per_row, sc, s[i]);
      }
    }
  }
}

// Rows of up to CAP columns through LDS.
template <typename T, int OUT, int VEC, int CAP>
__device__ __forceinline__ void rms_wide_body(const vrs_rms_args& a) {
  constexpr int NT = 1024;
  __shared__ __attribute__((aligned(16))) float s[CAP];     // a thread reads what it wrote alone
  __shared__ double lds_d[NT / 64];
  float* lds = reinterpret_cast<float*>(lds_d);
  const int c0 = threadIdx.x * VEC, step = NT * VEC;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    const T* res = a.res ? static_cast<const T*>(a.res) + row * a.res_ld : nullptr;
    T* sum = a.sum ? static_cast<T*>(a.sum) + row * a.sum_ld : nullptr;
    float ss = 0.f;
    for (int c = c0; c < a.cols; c += step) {
      float v[VEC];
      Raw<T, VEC> u;
      u.load(x + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = u[e];
      if (res) {
        u.load(res + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += u[e];
      }
      if (sum) store_vec<T, VEC>(sum + c, v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[c + e] = v[e];
        ss += v[e] * v[e];
      }
    }
    ss = row_reduce<float, NT, false>(ss, lds);
    float r;
    if (in_range(ss)) {
      r = 1.f / sqrtf(ss / (float)a.cols + a.eps);
    } else {     // the same sum in 64 bits
      double sd = 0.0;
      for (int c = c0; c < a.cols; c += step)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sd += (double)s[c + e] * (double)s[c + e];
      sd = row_reduce<double, NT, false>(sd, lds_d);
      r = (float)(1.0 / sqrt(sd / (double)a.cols + (double)a.eps));
    }
    auto value = [&](int c, float (&y)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[e] = c < a.cols ? s[c + e] * r * a.weight[c + e] : 0.f;
    };
    if constexpr (OUT == kSame) {
      for (int c = c0; c < a.cols; c += step) {
        float y[VEC];
        value(c, y);
        store_vec<T, VEC>(static_cast<T*>(a.y) + row * a.y_ld + c, y);
      }
    } else {
      Scale sc = Scale::step(a.inv_step);
      const bool per_row = a.group == a.cols;
      if (per_row) {
        float amax = 0.f;
        for (int c = c0; c < a.cols; c += step) {
          float y[VEC];
          value(c, y);
#pragma unroll
          for (int e = 0; e < VEC; ++e) amax = fmaxf(amax, fabsf(y[e]));
        }
        sc = Scale::of(row_reduce<float, NT, true>(amax, lds));
        if (threadIdx.x == 0) a.scales[row] = sc.scale;
      }
      for (int b = 0; b < a.cols; b += step) {     // every lane to the end: a group's lanes meet
        float y[VEC];
        value(b + c0, y);
        put_fp8<VEC>(a, row, b + c0, b + c0 < a.cols, per_row, sc, y);
      }
    }
  }
}
}  // namespace

#define VRS_RMS(TN, T, ON, OUT, TPR, NV, VEC)                                                          \
  extern "C" __global__ __launch_bounds__(256) void vrs_rms_##TN##_##ON##_##TPR##x##NV##_v##VEC( \
      vrs_rms_args a) {                                                                                \
    rms_body<T, OUT, TPR, NV, VEC>(a);                                                                 \
  }
#define VRS_RMS_WIDE(TN, T, ON, OUT, VEC)                                                               \
  extern "C" __global__ __launch_bounds__(1024) void vrs_rms_##TN##_##ON##_wide16k_v##VEC(vrs_rms_args a) { \
    rms_wide_body<T, OUT, VEC, 16384>(a);                                                               \
  }                                                                                                     \
  extern "C" __global__ __launch_bounds__(1024) void vrs_rms_##TN##_##ON##_wide32k_v##VEC(vrs_rms_args a) { \
    rms_wide_body<T, OUT, VEC, 32768>(a);                                                               \
  }
#define VRS_RMS_OUT(TN, T, ON, OUT, VEC)  \
  VRS_RMS(TN, T, ON, OUT, 64, 1, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 64, 2, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 64, 4, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 256, 2, VEC)    \
  VRS_RMS(TN, T, ON, OUT, 256, 4, VEC)    \
  VRS_RMS_WIDE(TN, T, ON, OUT, VEC)
VRS_RMS_OUT(bf16, bf16_t, same, kSame, 8)
VRS_RMS_OUT(bf16, bf16_t, e4m3, kFp8, 8)
VRS_RMS_OUT(f32, float, same, kSame, 4)
VRS_RMS_OUT(f32, float, e4m3, kFp8, 4)
// rows that no 16-byte vector divides, one element at a time
#define VRS_RMS_ONE(TN, T)                \
  VRS_RMS(TN, T, same, kSame, 64, 4, 1)   \
  VRS_RMS(TN, T, same, kSame, 256, 4, 1)  \
  VRS_RMS_WIDE(TN, T, same, kSame, 1)
VRS_RMS_ONE(bf16, bf16_t)
VRS_RMS_ONE(f32, float)
