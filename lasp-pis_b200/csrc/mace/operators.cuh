// Device helpers of the dense layer and layer norm: element types, activations, the column
// sum's second stage.
#pragma once
#include "operators.hpp"
#include "../lapis/launch.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstring>

namespace mace {
namespace op {
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// U neighbouring elements, moved by one load or store.
template <class T, int U> struct alignas(sizeof(T) * U) Unit {
  T v[U];
};
// Two 16-bit elements of one word.
__device__ __forceinline__ float2 to_floats(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 to_floats(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t to_word(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t to_word(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// A unit to floats and back, whole words at a time.
template <class T, int U> __device__ __forceinline__ void unpack(const Unit<T, U> &u, float *v) {
  if constexpr (sizeof(T) == 2 && U > 1) {
    uint32_t w[U / 2];
    memcpy(w, &u, sizeof u);
#pragma unroll
    for (int i = 0; i < U / 2; ++i) {
      const float2 f = to_floats(T{}, w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i)
      v[i] = to_float(u.v[i]);
  }
}
template <class T, int U> __device__ __forceinline__ Unit<T, U> pack(const float *v) {
  Unit<T, U> u;
  if constexpr (sizeof(T) == 2 && U > 1) {
    uint32_t w[U / 2];
#pragma unroll
    for (int i = 0; i < U / 2; ++i)
      w[i] = to_word(T{}, v[2 * i], v[2 * i + 1]);
    memcpy(&u, w, sizeof u);
  } else {
#pragma unroll
    for (int i = 0; i < U; ++i)
      u.v[i] = from_float<T>(v[i]);
  }
  return u;
}

// exp(-|z|): SiLU and its slope by quotients over 1 + exp(-|z|), in [1, 2], where nothing overflows and the
// fast division (2 ulp; the exact one branches for every value) has no range in which it gives 0.  16-bit
// results take the fast exponential (2^-21 of the value and a little more for large |z|, far below
// their own rounding).
template <bool Fast> __device__ __forceinline__ float exp_minus_abs(float z) {
  return Fast ? __expf(-fabsf(z)) : expf(-fabsf(z));
}
// Phi(-m) for m >= 0, as exp(-m^2 / 2) g(m): g, a scaled complementary error function, is a polynomial
// in t = 1 / (1 + 0.32 m), fitted here for the least relative error (4.4e-7).  e: the exponential.
// For 16-bit results (15 instructions, no branch; erff takes twice that).
__device__ __forceinline__ float normal_tail(float m, float &e) {
  const float t = __fdividef(1.f, fmaf(0.32f, m, 1.f));
  e = __expf(-0.5f * m * m);
  float q = 0.03452073782682419f;
  q = fmaf(q, t, -0.12243109941482544f);
  q = fmaf(q, t, 0.10611509531736374f);
  q = fmaf(q, t, 0.015589500777423382f);
  q = fmaf(q, t, 0.09737381339073181f);
  q = fmaf(q, t, 0.11343884468078613f);
  q = fmaf(q, t, 0.12773342430591583f);
  q = fmaf(q, t, 0.1276599019765854f);
  return q * t * e;
}
template <bool Fast> __device__ __forceinline__ float activate(float z, int act) {
  if (act == Silu) {
    const float e = exp_minus_abs<Fast>(z);
    return __fdividef(z < 0.f ? z * e : z, 1.f + e);
  }
  if (act == Gelu && Fast) { // z Phi(z) = max(z, 0) - |z| Phi(-|z|); the tail is 0 from 40 on, NaN stays
    const float m = fmaxf(-z, fminf(z, 40.f)); // |z|; the formula's NaN for -infinity, but not for infinity
    float e;
    return fmaf(-m, normal_tail(m, e), z < 0.f ? 0.f : z);
  }
  if (act == Gelu)
    return 0.5f * z * (1.f + erff(z * 0.70710678f));
  if (act == Relu)
    return z < 0.f ? 0.f : z; // NaN stays
  return z;
}
// N values at once: one branch on the activation, so that the values' arithmetic interleaves.
template <bool Fast, int N> __device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  if (act == Silu) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = activate<Fast>(v[i], Silu);
  } else if (act == Gelu) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = activate<Fast>(v[i], Gelu);
  } else if (act == Relu) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = activate<Fast>(v[i], Relu);
  }
}
// d act / dz
template <bool Fast> __device__ __forceinline__ float slope(float z, int act) {
  if (act == Silu) {
    const float e = exp_minus_abs<Fast>(z), s = __fdividef(z < 0.f ? e : 1.f, 1.f + e);
    return s * (1.f + z * (1.f - s));
  }
  if (act == Gelu && Fast) {
    const float m = fminf(fabsf(z), 40.f);
    float e;
    const float h = normal_tail(m, e), s = fmaf(copysignf(m, z), e * 0.39894228f, z < 0.f ? h : 1.f - h);
    return fmaf(z, 0.f, s); // NaN where z is not finite, as the formula
  }
  if (act == Gelu) {
    float e = expf(-0.5f * z * z);
    return 0.5f * (1.f + erff(z * 0.70710678f)) + z * e * 0.39894228f;
  }
  if (act == Relu)
    return z <= 0.f ? 0.f : 1.f; // NaN passes the gradient, as a comparison that fails
  return 1.f;
}
// The slopes of N values in their place.
template <bool Fast, int N> __device__ __forceinline__ void slope_all(float (&v)[N], int act) {
  if (act == Silu) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = slope<Fast>(v[i], Silu);
  } else if (act == Gelu) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = slope<Fast>(v[i], Gelu);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = slope<Fast>(v[i], act);
  }
}

// Second stage of a sum over rows: out_k[c] = sum over p < parts of partial[p][k][c], k < 2
// (out_k NULL: skipped), in a fixed order: lane group y takes p = y, y + 32, ..., then a tree.
// 32 columns per block; the partials come from L2, so latency bounds it.
template <class T> __global__ void __launch_bounds__(1024) column_sum_kernel(const float *partial, int parts, int planes,
                                                                             long long width, T *out0, T *out1) {
  __shared__ float sum[32][33];
  int x = threadIdx.x & 31, y = threadIdx.x >> 5, k = blockIdx.y;
  long long c = (long long)blockIdx.x * 32 + x;
  T *out = k ? out1 : out0;
  if (!out)
    return;
  float s = 0.f;
  if (c < width)
    for (int p = y; p < parts; p += 32)
      s += partial[((long long)p * planes + k) * width + c];
  sum[y][x] = s;
  __syncthreads();
  float v = sum[x][y]; // warp y sums column y over its lanes
#pragma unroll
  for (int o = 16; o; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  c = (long long)blockIdx.x * 32 + y;
  if (!x && c < width)
    out[c] = from_float<T>(v);
}

// SMs of the current device (148, a B200's, on a host without one: sizes can be asked there).
inline int sm_count() {
  static thread_local int device = -1, sms = 148;
  int now = 0;
  if (cudaGetDevice(&now) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  if (now != device) {
    lapis::check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, now));
    device = now;
  }
  return sms;
}
inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
template <class F> void with_type(int type, F &&f) {
  if (type == F32)
    f(float{});
  else if (type == BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}
} // namespace op
} // namespace mace
