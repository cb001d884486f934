// Shared by the fp32 window attention kernels for training (attention_grad_simt.cu,
// attention_grad_tf32.cu): their parameters, loads, bias and mask.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace crumpet {
namespace grad_f32 {

constexpr float kLog2e = 1.4426950408889634f;
enum Mode { kForward, kRows, kCols };

struct Params {
  const void* qkv;    // [B, N, 3, H, D]
  const void* dout;   // [B, N, H, D]
  void* dqkv;         // [B, N, 3, H, D]
  float* dbias;       // [S, H, N, N]
  float2* stats;      // [B, H, N]
  const void* table;  // [T, H]
  const int* pairs;   // [N, N]
  int table_f32, table_rows, analytic;
  int* error;         // training_error_word
  int nwd, nwh, nww, wsd, wsh, wsw, ssd, ssh, ssw;
  int B, H, N, QB, S, bias_pitch;
  int vec;            // every tensor on 16-byte boundaries: four channels per load
  float scale;
  void* out;          // forward: [B, N, H, D]
};

template <typename T>
__device__ __forceinline__ float load(const T* p, long long i);
template <>
__device__ __forceinline__ float load<float>(const float* p, long long i) { return __ldg(p + i); }
template <>
__device__ __forceinline__ float load<__half>(const __half* p, long long i) {
  return __half2float(__ldg(p + i));
}
template <>
__device__ __forceinline__ float load<__nv_bfloat16>(const __nv_bfloat16* p, long long i) {
  return __bfloat162float(__ldg(p + i));
}
template <typename T>
__device__ __forceinline__ T store_as(float v);
template <>
__device__ __forceinline__ float store_as<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half store_as<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 store_as<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t side_code(const Params& p, int t) {
  const int lw = t % p.wsw, t2 = t / p.wsw;
  const int lh = t2 % p.wsh, ld = t2 / p.wsh;
  return uint32_t(ld >= p.wsd - p.ssd) | (uint32_t(lh >= p.wsh - p.ssh) << 1) |
         (uint32_t(lw >= p.wsw - p.ssw) << 2);
}
__device__ __forceinline__ uint32_t last_axes(const Params& p, int b) {
  if (!p.analytic) return 0;
  const int wi = b % (p.nwd * p.nwh * p.nww);
  const int iw = wi % p.nww, t = wi / p.nww;
  const int ih = t % p.nwh, id = t / p.nwh;
  return uint32_t(p.ssd != 0 && id == p.nwd - 1) | (uint32_t(p.ssh != 0 && ih == p.nwh - 1) << 1) |
         (uint32_t(p.ssw != 0 && iw == p.nww - 1) << 2);
}

// Four consecutive channels as fp32
template <typename T>
__device__ __forceinline__ float4 load4(const Params& p, const T* at) {
  if (p.vec) {
    if constexpr (sizeof(T) == 4) {
      return __ldg(reinterpret_cast<const float4*>(at));
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(at));
      const T* v = reinterpret_cast<const T*>(&w);
      return make_float4(float(v[0]), float(v[1]), float(v[2]), float(v[3]));
    }
  }
  return make_float4(load(at, 0), load(at, 1), load(at, 2), load(at, 3));
}

// A bucket read from `pairs`, and the largest one read
__device__ __forceinline__ unsigned bucket_of(const Params& p, long long pair, unsigned& most) {
  const unsigned t = unsigned(__ldg(p.pairs + pair));
  most = max(most, t);
  return t;
}
__device__ __forceinline__ void check_buckets(const Params& p, unsigned most) {
  if (most >= unsigned(p.table_rows)) atomicOr(p.error, 2);
}
// bias of one bucket times log2 e; 0 (a clamped load's place) outside the table
template <typename T>
__device__ __forceinline__ float bias_of(const Params& p, int h, unsigned t) {
  const long long at = (long long)min(t, unsigned(p.table_rows) - 1) * p.H + h;
  const float v = kLog2e * (p.table_f32 ? __ldg(static_cast<const float*>(p.table) + at)
                                        : load(static_cast<const T*>(p.table), at));
  return t < unsigned(p.table_rows) ? v : 0.f;
}

// Allows a kernel `bytes` of dynamic shared memory on the current device, once: the most that any
// call takes.  (Set to each call's own size, one thread would lower it between another's call and
// its launch.)  `allowed` is the kernel's own, per device.
template <class K>
int allow_smem(K kernel, int bytes, std::atomic<bool> (&allowed)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && allowed[dev].load(std::memory_order_acquire)) return kOk;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return set_cuda_error(e, "attention (fp32) smem attribute");
  if (dev < 64) allowed[dev].store(true, std::memory_order_release);
  return kOk;
}

}  // namespace grad_f32

// attention_grad_tf32.cu: fp32 tensors, head_dim 16 or 32
inline bool attention_tf32(int dtype, int64_t head_dim) { return dtype == kF32 && head_dim <= 32; }
int64_t attention_grad_shares_tf32(int64_t B, int64_t H, int64_t N);
int launch_attention_tf32(const grad_f32::Params& p, int head_dim, bool forward,
                          cudaStream_t stream);

}  // namespace crumpet
