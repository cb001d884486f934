// crumpet_b200: GELU whose input is kept in 8 bits for the backward pass.
//
// The MLP's backward needs gelu'(u) for the input's gradient and gelu(u) again for the second
// Linear's weight gradient.  Instead of u and gelu(u) (4 bytes per element in 16-bit training)
// one byte is kept: per 32 neighbouring channels of a row the least power of two s = 2^e with
// max|u| <= 127 s (one byte, e + 127), and q = rint(u / s) as int8.  A power of two makes u / s
// and q s exact, so what is kept does not depend on how it is computed, and lets one byte serve
// 32 channels (an fp32 scale would take 12.5 %); it costs up to one of the 8 bits.  In a group
// whose largest value would be read back as 64 s = 2^128 (2^16 in fp16), an infinity, |q| stops at
// 63, so what is finite reads back finite.  A group that
// holds an infinity or NaN has scale byte 255 and q = 0, which reads back as NaN, so an
// overflowed step is seen in the gradients.
//
// GELU(u) = u F(u), GELU'(u) = F(u) + u f(u), with the normal distribution's F and density f:
// F(-|u|) = erfc(|u| / sqrt 2) / 2 by Abramowitz & Stegun, Handbook of Mathematical Functions,
// formula 7.1.26 (|error| <= 1.5e-7 in erf, so 0.75e-7 |u| in GELU; in the tail that is part of a
// small value: 5e-5 of it at -3, 1e-2 at -8), one reciprocal, one exponential (shared with f) and five
// FMAs.
//
// HBM traffic bounds both kernels: 5 bytes per element forward and 7 backward in 16 bits.  Four
// lanes share a group (8 elements each, 16-byte accesses).
//
// Measured: 442368 x 192 in bf16, 81 us forward (66 us of HBM time; issue slots 77 % busy) and
// 109 us backward (92 us).  The forward loads a group ahead; the backward, which has more CTAs in
// flight, lost by that (108 us).
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
__device__ __forceinline__ void load8(const T* p, Pack8<T>& w) {
#pragma unroll
  for (int k = 0; k < int(sizeof(w)) / 16; ++k)
    reinterpret_cast<uint4*>(&w)[k] = ldg_stream(reinterpret_cast<const uint4*>(p) + k);
}
template <typename T>
__device__ __forceinline__ void unpack8(const Pack8<T>& w, float (&x)[8]) {
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

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// max(x, 0), NaN for NaN
__device__ __forceinline__ float relu(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}

// F(-|x|) of two values, and exp(-x^2 / 2) in *e; the packed arithmetic takes two per instruction
__device__ __forceinline__ float2 lower_tail(float2 a, float2* e) {
  // a = |x|: 1 + 0.3275911 a / sqrt 2, and -a^2 / 2 in powers of two
  const float2 d = __ffma2_rn(a, both(0.23164189f), both(1.f));
  const float2 y = __fmul2_rn(__fmul2_rn(a, a), both(-0.72134752044448170f));
  float2 t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t.y) : "f"(d.y));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e->x) : "f"(y.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e->y) : "f"(y.y));
  // half the formula's coefficients: F(-a) = erfc / 2
  float2 q = __ffma2_rn(both(0.5307027145f), t, both(-0.7265760135f));
  q = __ffma2_rn(q, t, both(0.7107068705f));
  q = __ffma2_rn(q, t, both(-0.142248368f));
  q = __ffma2_rn(q, t, both(0.127414796f));
  return __fmul2_rn(__fmul2_rn(q, t), *e);
}
// gelu(x) = x F(x) = max(x, 0) - |x| F(-|x|): one expression for both signs; the
// infinite ends are exact.  |x| is taken as finite, so infinities give inf and 0; NaN gives NaN through max(x, 0).
__device__ __forceinline__ float2 gelu(float2 x) {
  constexpr float kMax = 3.402823466e38f;
  const float2 a = make_float2(fminf(fabsf(x.x), kMax), fminf(fabsf(x.y), kMax));
  float2 e;
  const float2 q = lower_tail(a, &e);
  return __ffma2_rn(make_float2(-a.x, -a.y), q, make_float2(relu(x.x), relu(x.y)));
}
// gelu and its slope F(x) + x f(x) of finite x or NaN: with r = |x| f - F(-|x|) the slope is 1 + r,
// and -r for negative x
__device__ __forceinline__ float2 gelu_slope(float2 x, float2* y) {
  const float2 a = make_float2(fabsf(x.x), fabsf(x.y));
  float2 e;
  const float2 q = lower_tail(a, &e);
  *y = __ffma2_rn(make_float2(-a.x, -a.y), q, make_float2(relu(x.x), relu(x.y)));
  const float2 r = __ffma2_rn(__fmul2_rn(a, both(0.39894228040143268f)), e,
                              make_float2(-q.x, -q.y));
  const float2 s = make_float2(copysignf(1.f, x.x), copysignf(1.f, x.y));
  return __ffma2_rn(r, s, __ffma2_rn(s, both(0.5f), both(0.5f)));
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

// The scale byte whose 64 s overflows the element type (rounding reaches 64 there at most); the
// only one above it is 255.
template <typename T>
constexpr uint32_t kTopCode = 249u;
template <>
constexpr uint32_t kTopCode<__half> = 137u;

// Rounding to whole numbers by adding 1.5 * 2^23: the sum's low byte is q in two's complement.
// In a group with an infinity or NaN (code 255) q is 0.
constexpr float kRound = 12582912.f;
__device__ __forceinline__ uint32_t low_bytes(const uint32_t (&b)[4]) {
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}
template <typename T>
__device__ __forceinline__ uint32_t quantise4(const float* x, float inv, uint32_t code) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(x[i], inv, kRound));
  if (code >= kTopCode<T>) {
    if (code == 255u) return 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = __float_as_uint(fminf(fmaxf(__uint_as_float(b[i]), kRound - 63.f), kRound + 63.f));
  }
  return low_bytes(b);
}
template <typename T>
__device__ __forceinline__ int quantise(float x, float inv, uint32_t code) {
  if (code == 255u) return 0;
  if (code == kTopCode<T>) return int(fminf(fmaxf(rintf(x * inv), -63.f), 63.f));
  return int(int8_t(__float_as_uint(fmaf(x, inv, kRound)) & 0xffu));
}
// u of four values of a word: a byte with its sign bit flipped, under the exponent of 2^23, is
// 2^23 + 128 + q
__device__ __forceinline__ void restore4(uint32_t w, float s, float* x) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440u + i)) - 8388736.f) * s;
}

struct Rows {
  bool whole;           // rows of whole groups: group g holds elements [32 g, 32 g + 32)
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

// Where the 8 channels of part `part` of a group lie
struct Place {
  long long at;
  bool in_group, in;
};
__device__ __forceinline__ Place find_part(const Rows& r, long long grp, int part) {
  Place q;
  q.in_group = grp < r.groups;
  if (r.whole) {
    q.in = q.in_group;
    q.at = grp * kGroup + part * 8;
    return q;
  }
  long long row = 0;
  int c = 0;
  if (q.in_group) place(r, grp, &row, &c);
  c += part * 8;
  q.in = q.in_group && c < r.C;
  q.at = row * r.C + c;
  return q;
}

// C a multiple of 8 and 16-byte aligned tensors: four lanes per group
template <typename T>
__global__ void __launch_bounds__(kThreads)
gelu_keep_kernel(T* y, int8_t* kept, uint8_t* scales, const T* x, Rows r) {
  const int part = threadIdx.x & 3;
  const long long step = (long long)gridDim.x * (kThreads / 4);
  auto find = [&](long long grp) { return find_part(r, grp, part); };
  long long grp = blockIdx.x * (long long)(kThreads / 4) + (threadIdx.x >> 2);
  // the next group's load is in flight through this one's arithmetic
  Place q = find(grp);
  Pack8<T> ahead = {};
  if (q.in) load8(x + q.at, ahead);
  // whole warps take part in the shuffles: the bound is rounded up to a warp's 8 groups
  for (; grp - (grp & 7) < r.groups; grp += step) {
    const long long at = q.at;
    const bool in_group = q.in_group, in = q.in;
    float v[8] = {};
    if (in) unpack8(ahead, v);
    q = find(grp + step);
    if (q.in) load8(x + q.at, ahead);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    const uint32_t code = scale_code(top);
    if (in_group && part == 0) scales[grp] = uint8_t(code);
    if (!in) continue;
    const float inv = code_inverse(code);
    stg(reinterpret_cast<uint2*>(kept + at),
        make_uint2(quantise4<T>(v, inv, code), quantise4<T>(v + 4, inv, code)));
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float2 f = gelu(make_float2(v[i], v[i + 1]));
      v[i] = f.x;
      v[i + 1] = f.y;
    }
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
      kept[at] = int8_t(quantise<T>(v, code_inverse(code), code));
      y[at] = from_f32<T>(gelu(both(v)).x);
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
    const Place q = find_part(r, grp, part);
    if (!q.in) continue;
    const long long at = q.at;
    const uint2 w = ldg_stream(reinterpret_cast<const uint2*>(kept + at));
    Pack8<T> gw;
    if constexpr (GRAD) load8(grad_y + at, gw);
    const float s = code_step(__ldg(scales + grp));
    float a[8];
    restore4(w.x, s, a);
    restore4(w.y, s, a + 4);
    float g[8];
    if constexpr (GRAD) {
      unpack8(gw, g);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float2 y;
        const float2 slope = gelu_slope(make_float2(a[i], a[i + 1]), &y);
        g[i] *= slope.x;
        g[i + 1] *= slope.y;
        a[i] = y.x;
        a[i + 1] = y.y;
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
      float2 y;
      const float slope = gelu_slope(both(x), &y).x;
      grad_x[at] = from_f32<T>(to_f32(grad_y[at]) * slope);
      again[at] = from_f32<T>(y.x);
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
  r.whole = C % kGroup == 0;
  r.groups = M * int64_t(r.per_row);
  r.div = DivMod32::make(r.per_row);
  r.C = int(C);
  return r;
}

unsigned grid_for(int64_t groups, int per_block, int per_sm) {
  const int64_t want = (groups + per_block - 1) / per_block;
  const int64_t most = int64_t(sm_count()) * per_sm;
  return unsigned(want < most ? want : most);
}

template <typename T>
int keep(void* y, int8_t* kept, uint8_t* scales, const void* x, int64_t M, int64_t C,
         cudaStream_t stream) {
  const Rows r = make_rows(M, C);
  if (C % 8 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(kept, 8))
    gelu_keep_kernel<T><<<grid_for(r.groups, kThreads / 4, 16), kThreads, 0, stream>>>(
        static_cast<T*>(y), kept, scales, static_cast<const T*>(x), r);
  else
    gelu_keep_any_kernel<T><<<grid_for(r.groups, kThreads / 32, 64), kThreads, 0, stream>>>(
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
    kept_use_kernel<T, GRAD><<<grid_for(r.groups, kThreads / 4, 64), kThreads, 0, stream>>>(
        static_cast<T*>(grad_x), static_cast<T*>(again), static_cast<const T*>(grad_y), kept,
        scales, r);
  else
    kept_use_any_kernel<T, GRAD><<<grid_for(r.groups, kThreads / 32, 64), kThreads, 0, stream>>>(
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
