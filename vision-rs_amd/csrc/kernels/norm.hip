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
// registers.  Wide rows take more threads, not more registers.
#include "common.h"

namespace {
constexpr int kSame = 0, kFp8 = 1;
constexpr float kE4m3Max = 448.f;

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&o)[VEC]) {
  if constexpr (VEC == 1) {
    o[0] = Elt<T>::to_f(*p);
  } else {
    static_assert(VEC * sizeof(T) == 16, "one 16-byte load");
    const u32x4_t u = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        o[i] = __uint_as_float(u[i]);
      } else {
        o[2 * i] = __uint_as_float(u[i] << 16);
        o[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
}
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

template <typename T, int OUT, int TPR, int NV, int VEC>
__device__ __forceinline__ void rms_body(const vrs_rms_args& a) {
  constexpr int WG = TPR < 256 ? 256 : TPR, RPW = WG / TPR;   // rows per workgroup step
  __shared__ double lds_d[WG / 64];
  float* lds = reinterpret_cast<float*>(lds_d);
  const int t = threadIdx.x % TPR;
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.res);
  T* sum = static_cast<T*>(a.sum);

  // The next row's loads are in flight while this one is reduced and stored (8192 rows of 4096 in
  // bfloat16 with the residual: 50 us, 5.3 TB/s, against 58 without); not where 1024 threads hold a
  // row, whose registers are full.
  constexpr bool kAhead = TPR <= 256;
  float w[NV][VEC];      // the weights of this thread's columns, held likewise
  auto weight = [&](int i) {
    const int c = (i * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[i][e] = c < a.cols ? a.weight[c + e] : 0.f;
  };
  if constexpr (kAhead) {
#pragma unroll
    for (int i = 0; i < NV; ++i) weight(i);
  }
  float nx[NV][VEC], nr[NV][VEC];
  auto fetch = [&](int64_t r0) {
    const int64_t row = r0 + threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (row < a.rows && c < a.cols) {
        load_vec<T, VEC>(x + row * a.x_ld + c, nx[i]);
        if (res) load_vec<T, VEC>(res + row * a.res_ld + c, nr[i]);
      }
    }
  };
  if constexpr (kAhead) fetch((int64_t)blockIdx.x * RPW);
  // every thread of a workgroup makes every step (the reductions of wide rows have barriers)
  for (int64_t r0 = (int64_t)blockIdx.x * RPW; r0 < a.rows; r0 += (int64_t)gridDim.x * RPW) {
    if constexpr (!kAhead) fetch(r0);
    const int64_t row = r0 + threadIdx.x / TPR;
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
    if constexpr (kAhead) fetch(r0 + (int64_t)gridDim.x * RPW);
    ss = row_reduce<float, TPR, false>(ss, lds);
    float r;
    if (ss > 1e-25f && ss < INFINITY) {
      r = 1.f / sqrtf(ss / (float)a.cols + a.eps);
    } else {
      // squares below or above float32's range (or a NaN): the same sum in 64 bits
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
    for (int i = 0; i < NV; ++i) {
      if constexpr (!kAhead) weight(i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[i][e] = s[i][e] * r * w[i][e];
        if constexpr (OUT == kFp8) amax = fmaxf(amax, fabsf(s[i][e]));
      }
    }
    if constexpr (OUT == kSame) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (ok && c < a.cols) store_vec<T, VEC>(static_cast<T*>(a.y) + row * a.y_ld + c, s[i]);
      }
    } else {
      float inv = a.inv_step;
      const bool per_row = a.group == a.cols;
      if (per_row) {
        amax = row_reduce<float, TPR, true>(amax, lds);
        inv = amax > 0.f ? kE4m3Max / amax : 1.f;
        if (ok && t == 0) a.scales[row] = amax > 0.f ? amax / kE4m3Max : 1.f;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (a.group && !per_row) {     // lanes of one group are neighbours in a wave
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < VEC; ++e) m = fmaxf(m, fabsf(s[i][e]));
          const int lanes = a.group / VEC;
          for (int d = 1; d < lanes; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
          inv = m > 0.f ? kE4m3Max / m : 1.f;
          if (ok && c < a.cols && c % a.group == 0)
            a.scales[row * (a.cols / a.group) + c / a.group] = m > 0.f ? m / kE4m3Max : 1.f;
        }
        if (ok && c < a.cols) {
          float q[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) q[e] = s[i][e] * inv;
          store_fp8<VEC>(static_cast<uint8_t*>(a.y) + row * a.y_ld + c, q);
        }
      }
    }
  }
}
}  // namespace

#define VRS_RMS(TN, T, ON, OUT, TPR, NV, VEC)                                                          \
  extern "C" __global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void vrs_rms_##TN##_##ON##_##TPR##x##NV##_v##VEC( \
      vrs_rms_args a) {                                                                                \
    rms_body<T, OUT, TPR, NV, VEC>(a);                                                                 \
  }
#define VRS_RMS_OUT(TN, T, ON, OUT, VEC)  \
  VRS_RMS(TN, T, ON, OUT, 64, 1, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 64, 2, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 64, 4, VEC)     \
  VRS_RMS(TN, T, ON, OUT, 256, 2, VEC)    \
  VRS_RMS(TN, T, ON, OUT, 256, 4, VEC)    \
  VRS_RMS(TN, T, ON, OUT, 1024, 2, VEC)   \
  VRS_RMS(TN, T, ON, OUT, 1024, 4, VEC)
VRS_RMS_OUT(bf16, bf16_t, same, kSame, 8)
VRS_RMS_OUT(bf16, bf16_t, e4m3, kFp8, 8)
VRS_RMS_OUT(f32, float, same, kSame, 4)
VRS_RMS_OUT(f32, float, e4m3, kFp8, 4)
VRS_RMS(f32, float, same, kSame, 1024, 8, 4)
VRS_RMS(f32, float, e4m3, kFp8, 1024, 8, 4)
// rows that no 16-byte vector divides, one element at a time
#define VRS_RMS_ONE(TN, T)                \
  VRS_RMS(TN, T, same, kSame, 64, 4, 1)   \
  VRS_RMS(TN, T, same, kSame, 256, 4, 1)  \
  VRS_RMS(TN, T, same, kSame, 256, 16, 1) \
  VRS_RMS(TN, T, same, kSame, 1024, 32, 1)
VRS_RMS_ONE(bf16, bf16_t)
VRS_RMS_ONE(f32, float)
