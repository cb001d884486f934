// crumpet_b200: GELU whose input is kept in 8 bits for the backward pass.
//
// The MLP's backward needs gelu'(u) for the input's gradient and gelu(u) again for the second
// Linear's weight gradient.  Instead of u and gelu(u) (4 bytes per element in 16-bit training)
// one byte is kept: per 32 neighbouring channels of a row the least power of two s = 2^e with
// max|u| <= 127 s (one byte, e + 127), and q = rint(u / s) as int8.  A power of two makes u / s
// and q s exact, so what is kept does not depend on how it is computed, and lets one byte serve
// 32 channels (an fp32 scale would take 12.5 %); it costs up to one of the 8 bits.  A group that
// holds an infinity or NaN has scale byte 255 and q = 0, which reads back as NaN, so an
// overflowed step is seen in the gradients.
//
// GELU(u) = u F(u), GELU'(u) = F(u) + u f(u), with the normal distribution's F and density f:
// F(-|u|) = erfc(|u| / sqrt 2) / 2 by Abramowitz & Stegun, Handbook of Mathematical Functions,
// formula 7.1.26 (|error| <= 1.5e-7 in erf), one reciprocal, one exponential (shared with f) and
// five FMAs.
//
// HBM traffic bounds both kernels: 5 bytes per element forward and 7 backward in 16 bits.  Four
// lanes share a group (8 elements each, 16-byte accesses).
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

constexpr int kGroup = 32;
constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T>
struct alignas(16) Pack8 {
  T v[8];
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  Pack8<T> w;
#pragma unroll
  for (int k = 0; k < int(sizeof(w)) / 16; ++k)
    reinterpret_cast<uint4*>(&w)[k] = ldg_stream(reinterpret_cast<const uint4*>(p) + k);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(w.v[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  Pack8<T> w;
#pragma unroll
  for (int i = 0; i < 8; ++i) w.v[i] = from_f32<T>(x[i]);
#pragma unroll
  for (int k = 0; k < int(sizeof(w)) / 16; ++k)
    stg(reinterpret_cast<uint4*>(p) + k, reinterpret_cast<const uint4*>(&w)[k]);
}

// F(x), and exp(-x^2 / 2) in *e
__device__ __forceinline__ float normal_cdf(float x, float* e) {
  const float z = fabsf(x) * 0.70710678118654752f;
  float t, ex;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f, z, 1.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ex) : "f"(z * z * -1.4426950408889634f));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  q = 0.5f * q * t * ex;  // F(-|x|)
  *e = ex;
  return x < 0.f ? q : 1.f - q;
}

// Scale byte of a group from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  // amax = m 2^k, 1 <= m < 2: 127 2^e reaches it from e = k - 6 while m <= 127 / 64
  const int e = int(amax_bits >> 23) - 127 - 6 + int((amax_bits & 0x7fffffu) > 0x7e0000u);
  return uint32_t(max(e, -126) + 127);
}
__device__ __forceinline__ float code_step(uint32_t code) { return __uint_as_float(code << 23); }
__device__ __forceinline__ float code_inverse(uint32_t code) {
  return __uint_as_float((code == 255u ? 0u : 254u - code) << 23);
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// q of one value: 0 in a group with an infinity or NaN (its inverse step is 0; the product of
// 0 and an infinity, NaN, converts to 0)
__device__ __forceinline__ int quantise(float x, float inv) { return __float2int_rn(x * inv); }

struct Rows {
  long long groups;     // rows x groups per row
  uint32_t per_row;     // groups per row
  DivMod32 div;         // by per_row (row and group from a 32-bit group number)
  int C;
};

__device__ __forceinline__ void place(const Rows& r, long long grp, long long* row, int* first) {
  long long q;
  if (r.groups <= 0xffffffffLL) {
    q = r.div.div(uint32_t(grp));
  } else {
    q = grp / r.per_row;
  }
  *row = q;
  *first = int(grp - q * r.per_row) * kGroup;
}

// C a multiple of 8 and 16-byte aligned tensors: four lanes per group
template <typename T>
__global__ void __launch_bounds__(kThreads)
gelu_keep_kernel(T* y, int8_t* kept, uint8_t* scales, const T* x, Rows r) {
  const int part = threadIdx.x & 3;
  const long long step = (long long)gridDim.x * (kThreads / 4);
  // whole warps take part in the shuffles: the bound is rounded up to a warp's 8 groups
  for (long long grp = blockIdx.x * (long long)(kThreads / 4) + (threadIdx.x >> 2);
       grp - (grp & 7) < r.groups; grp += step) {
    long long row = 0;
    int c = 0;
    const bool in_group = grp < r.groups;
    if (in_group) place(r, grp, &row, &c);
    c += part * 8;
    const bool in = in_group && c < r.C;
    const long long at = row * r.C + c;
    float v[8] = {};
    if (in) load8(x + at, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    const uint32_t code = scale_code(top);
    if (in_group && part == 0) scales[grp] = uint8_t(code);
    if (!in) continue;
    const float inv = code_inverse(code);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i >> 2] |= (uint32_t(quantise(v[i], inv)) & 0xffu) << (8 * (i & 3));
    stg(reinterpret_cast<uint2*>(kept + at), make_uint2(w[0], w[1]));
    float e;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= normal_cdf(v[i], &e);
    store8(y + at, v);
  }
}

// any width and alignment: a warp per group
template <typename T>
__global__ void __launch_bounds__(kThreads)
gelu_keep_any_kernel(T* y, int8_t* kept, uint8_t* scales, const T* x, Rows r) {
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (kThreads / 32);
  for (long long grp = blockIdx.x * (long long)(kThreads / 32) + (threadIdx.x >> 5);
       grp < r.groups; grp += step) {
    long long row;
    int c;
    place(r, grp, &row, &c);
    c += lane;
    const long long at = row * r.C + c;
    const float v = c < r.C ? to_f32(x[at]) : 0.f;
    const uint32_t code = scale_code(__reduce_max_sync(~0u, abs_bits(v)));
    if (lane == 0) scales[grp] = uint8_t(code);
    if (c < r.C) {
      kept[at] = int8_t(quantise(v, code_inverse(code)));
      float e;
      y[at] = from_f32<T>(v * normal_cdf(v, &e));
    }
  }
}

// GRAD: the input's gradient and the recomputed output; else the kept input itself.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads)
kept_use_kernel(T* grad_x, T* again, const T* grad_y, const int8_t* kept, const uint8_t* scales,
                Rows r) {
  const int part = threadIdx.x & 3;
  const long long step = (long long)gridDim.x * (kThreads / 4);
  for (long long grp = blockIdx.x * (long long)(kThreads / 4) + (threadIdx.x >> 2);
       grp < r.groups; grp += step) {
    long long row;
    int c;
    place(r, grp, &row, &c);
    c += part * 8;
    if (c >= r.C) continue;
    const long long at = row * r.C + c;
    const uint2 w = ldg_stream(reinterpret_cast<const uint2*>(kept + at));
    float g[8];
    if constexpr (GRAD) load8(grad_y + at, g);
    const float s = code_step(__ldg(scales + grp));
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = s * float(int8_t((i < 4 ? w.x : w.y) >> (8 * (i & 3))));
      if constexpr (GRAD) {
        float e;
        const float f = normal_cdf(x, &e);
        g[i] *= fmaf(x * 0.39894228040143268f, e, f);
        a[i] = x * f;
      } else {
        a[i] = x;
      }
    }
    if constexpr (GRAD) store8(grad_x + at, g);
    store8(again + at, a);
  }
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads)
kept_use_any_kernel(T* grad_x, T* again, const T* grad_y, const int8_t* kept,
                    const uint8_t* scales, Rows r) {
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * (kThreads / 32);
  for (long long grp = blockIdx.x * (long long)(kThreads / 32) + (threadIdx.x >> 5);
       grp < r.groups; grp += step) {
    long long row;
    int c;
    place(r, grp, &row, &c);
    c += lane;
    if (c >= r.C) continue;
    const long long at = row * r.C + c;
    const float x = code_step(__ldg(scales + grp)) * float(kept[at]);
    if constexpr (GRAD) {
      float e;
      const float f = normal_cdf(x, &e);
      grad_x[at] = from_f32<T>(to_f32(grad_y[at]) * fmaf(x * 0.39894228040143268f, e, f));
      again[at] = from_f32<T>(x * f);
    } else {
      again[at] = from_f32<T>(x);
    }
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

Rows make_rows(int64_t M, int64_t C) {
  Rows r{};
  r.per_row = uint32_t((C + kGroup - 1) / kGroup);
  r.groups = M * int64_t(r.per_row);
  r.div = DivMod32::make(r.per_row);
  r.C = int(C);
  return r;
}

unsigned grid_for(int64_t groups, int per_block) {
  const int64_t want = (groups + per_block - 1) / per_block;
  const int64_t most = int64_t(sm_count()) * 64;
  return unsigned(want < most ? want : most);
}

template <typename T>
int keep(void* y, int8_t* kept, uint8_t* scales, const void* x, int64_t M, int64_t C,
         cudaStream_t stream) {
  const Rows r = make_rows(M, C);
  if (C % 8 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(kept, 8))
    gelu_keep_kernel<T><<<grid_for(r.groups, kThreads / 4), kThreads, 0, stream>>>(
        static_cast<T*>(y), kept, scales, static_cast<const T*>(x), r);
  else
    gelu_keep_any_kernel<T><<<grid_for(r.groups, kThreads / 32), kThreads, 0, stream>>>(
        static_cast<T*>(y), kept, scales, static_cast<const T*>(x), r);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "gelu checkpoint launch");
}

template <typename T, bool GRAD>
int use(void* grad_x, void* again, const void* grad_y, const int8_t* kept, const uint8_t* scales,
        int64_t M, int64_t C, cudaStream_t stream) {
  const Rows r = make_rows(M, C);
  if (C % 8 == 0 && aligned(grad_x, 16) && aligned(again, 16) && aligned(grad_y, 16) &&
      aligned(kept, 8))
    kept_use_kernel<T, GRAD><<<grid_for(r.groups, kThreads / 4), kThreads, 0, stream>>>(
        static_cast<T*>(grad_x), static_cast<T*>(again), static_cast<const T*>(grad_y), kept,
        scales, r);
  else
    kept_use_any_kernel<T, GRAD><<<grid_for(r.groups, kThreads / 32), kThreads, 0, stream>>>(
        static_cast<T*>(grad_x), static_cast<T*>(again), static_cast<const T*>(grad_y), kept,
        scales, r);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "activation checkpoint launch");
}

}  // namespace

int launch_gelu_checkpoint(void* y, int8_t* kept, uint8_t* scales, const void* x, int dtype,
                           int64_t M, int64_t C, cudaStream_t stream) {
  if (dtype == kF32) return keep<float>(y, kept, scales, x, M, C, stream);
  if (dtype == kF16) return keep<__half>(y, kept, scales, x, M, C, stream);
  return keep<__nv_bfloat16>(y, kept, scales, x, M, C, stream);
}

int launch_gelu_checkpoint_backward(void* grad_x, void* again, const void* grad_y,
                                    const int8_t* kept, const uint8_t* scales, int dtype, int64_t M,
                                    int64_t C, cudaStream_t stream) {
  if (dtype == kF32) return use<float, true>(grad_x, again, grad_y, kept, scales, M, C, stream);
  if (dtype == kF16) return use<__half, true>(grad_x, again, grad_y, kept, scales, M, C, stream);
  return use<__nv_bfloat16, true>(grad_x, again, grad_y, kept, scales, M, C, stream);
}

int launch_restore_activation(void* x, const int8_t* kept, const uint8_t* scales, int dtype,
                              int64_t M, int64_t C, cudaStream_t stream) {
  if (dtype == kF32) return use<float, false>(nullptr, x, nullptr, kept, scales, M, C, stream);
  if (dtype == kF16) return use<__half, false>(nullptr, x, nullptr, kept, scales, M, C, stream);
  return use<__nv_bfloat16, false>(nullptr, x, nullptr, kept, scales, M, C, stream);
}

}  // namespace crumpet
