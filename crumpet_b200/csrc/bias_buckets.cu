// crumpet_b200: learned relative-position bias by buckets, and its gradient.
//
//   bias[h, i, j] = table[pairs[i, j], h]
//   grad_table[t, h] = sum over the pairs (i, j) of bucket t of grad[h, i, j]
//
// Both move one value per (head, pair) and compute next to nothing, so memory traffic and, at
// a Swin window's size (343 x 343 pairs), launch latency bound them.
//
// Forward: a CTA takes one head and a run of pairs.  The head's column of the table goes to
// shared memory first (2197 rows of a 7x7x7 window are 8.8 KB): neighbouring pairs have
// neighbouring buckets, so gathers from the transposed column meet few bank conflicts, where
// gathers from the [T, H] table would touch a 32-byte sector each.
//
// Gradient: no atomics, so the sum's order never changes.  The caller sorted the pairs by
// bucket once (`order`) and cut every bucket into items of a bounded number of pairs; one
// warp sums one (item, head), in a fixed order, in fp32.  The warps of a CTA take neighbouring
// items of one head, whose pairs are neighbours in memory, so the sectors that one gather
// opens serve the others from L1.  Buckets of several items are finished by a second kernel.
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 8;                  // pairs per thread of the forward kernel
constexpr int kTableSmem = 48 * 1024;          // largest table column kept in shared memory

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T, typename O, bool SMEM>
__global__ void __launch_bounds__(kThreads)
bias_gather_kernel(O* bias, const T* table, const int* pairs, long long npairs, int rows, int H) {
  extern __shared__ float column[];
  const int h = blockIdx.y;
  if constexpr (SMEM) {
    for (int t = threadIdx.x; t < rows; t += kThreads)
      column[t] = to_float(table[(long long)t * H + h]);
    __syncthreads();
  }
  O* out = bias + h * npairs;
  const long long step = (long long)kThreads * kPerThread;
  for (long long base = blockIdx.x * step; base < npairs; base += gridDim.x * step) {
    int t[kPerThread];
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) {
      const long long i = base + u * kThreads + threadIdx.x;
      t[u] = i < npairs ? __ldg(pairs + i) : 0;
    }
#pragma unroll
    for (int u = 0; u < kPerThread; ++u) {
      const long long i = base + u * kThreads + threadIdx.x;
      if (i < npairs)
        out[i] = from_float<O>(SMEM ? column[t[u]] : to_float(table[(long long)t[u] * H + h]));
    }
  }
}

struct GradBuckets {
  const int* order;      // [npairs] pairs sorted by bucket
  const int* items;      // [n_items][3]: bucket, begin, end (into order)
  const int* multi;      // [n_multi][3]: bucket, first item, last item + 1
  long long n_items, n_multi, npairs;
  int H;
};

// One warp per (item, head).  An item whose bucket is whole writes the table's gradient,
// the others their part of it: partial[item, h].
template <typename G, typename O>
__global__ void __launch_bounds__(kThreads)
bias_grad_kernel(O* grad_table, float* partial, const G* grad, int slabs, GradBuckets b) {
  const int lane = threadIdx.x & 31;
  const long long item = blockIdx.x * (long long)(kThreads / 32) + (threadIdx.x >> 5);
  const int h = blockIdx.y;
  if (item >= b.n_items) return;
  const int bucket = b.items[3 * item], begin = b.items[3 * item + 1], end = b.items[3 * item + 2];
  const long long slab = b.npairs * b.H;
  const G* src = grad + h * b.npairs;
  float sum = 0.f;
  for (int e = begin + lane; e < end; e += 32) {
    const long long at = b.order[e];
    for (int s = 0; s < slabs; ++s) sum += to_float(src[s * slab + at]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane != 0) return;
  if (bucket >= 0) grad_table[(long long)bucket * b.H + h] = from_float<O>(sum);
  else partial[item * b.H + h] = sum;
}

template <typename O>
__global__ void __launch_bounds__(kThreads)
bias_grad_join_kernel(O* grad_table, const float* partial, GradBuckets b) {
  const int lane = threadIdx.x & 31;
  const long long k = blockIdx.x * (long long)(kThreads / 32) + (threadIdx.x >> 5);
  const int h = blockIdx.y;
  if (k >= b.n_multi) return;
  const int bucket = b.multi[3 * k], first = b.multi[3 * k + 1], last = b.multi[3 * k + 2];
  float sum = 0.f;
  for (int i = first + lane; i < last; i += 32) sum += partial[(long long)i * b.H + h];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) grad_table[(long long)bucket * b.H + h] = from_float<O>(sum);
}

template <typename T, typename O>
int launch_gather(void* bias, const void* table, const int* pairs, int64_t npairs, int64_t rows,
                  int64_t H, cudaStream_t stream) {
  const int64_t step = int64_t(kThreads) * kPerThread;
  const int64_t want = (npairs + step - 1) / step;
  const dim3 grid(unsigned(want < 0x7fffffff ? want : 0x7fffffff), unsigned(H));
  if (rows * 4 <= kTableSmem)
    bias_gather_kernel<T, O, true><<<grid, kThreads, size_t(rows) * 4, stream>>>(
        static_cast<O*>(bias), static_cast<const T*>(table), pairs, npairs, int(rows), int(H));
  else
    bias_gather_kernel<T, O, false><<<grid, kThreads, 0, stream>>>(
        static_cast<O*>(bias), static_cast<const T*>(table), pairs, npairs, int(rows), int(H));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "relative position bias launch");
}

template <typename T>
int gather_out(void* bias, int out_dtype, const void* table, const int* pairs, int64_t npairs,
               int64_t rows, int64_t H, cudaStream_t stream) {
  if (out_dtype == kF32) return launch_gather<T, float>(bias, table, pairs, npairs, rows, H, stream);
  if (out_dtype == kF16)
    return launch_gather<T, __half>(bias, table, pairs, npairs, rows, H, stream);
  return launch_gather<T, __nv_bfloat16>(bias, table, pairs, npairs, rows, H, stream);
}

template <typename G, typename O>
int launch_grad(const BiasGradArgs& a, cudaStream_t stream) {
  GradBuckets b{a.order, a.items, a.multi, a.n_items, a.n_multi, a.npairs, int(a.H)};
  const int per = kThreads / 32;
  bias_grad_kernel<G, O><<<dim3(unsigned((a.n_items + per - 1) / per), unsigned(a.H)), kThreads, 0,
                           stream>>>(static_cast<O*>(a.grad_table), a.partial,
                                     static_cast<const G*>(a.grad), int(a.slabs), b);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "relative position bias gradient launch");
  if (a.n_multi > 0) {
    bias_grad_join_kernel<O><<<dim3(unsigned((a.n_multi + per - 1) / per), unsigned(a.H)),
                               kThreads, 0, stream>>>(static_cast<O*>(a.grad_table), a.partial, b);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "relative position bias gradient join launch");
  }
  return kOk;
}

template <typename G>
int grad_out(const BiasGradArgs& a, cudaStream_t stream) {
  if (a.table_dtype == kF32) return launch_grad<G, float>(a, stream);
  if (a.table_dtype == kF16) return launch_grad<G, __half>(a, stream);
  return launch_grad<G, __nv_bfloat16>(a, stream);
}

}  // namespace

int launch_relative_position_bias(void* bias, int out_dtype, const void* table, int table_dtype,
                                  const int* pairs, int64_t npairs, int64_t rows, int64_t H,
                                  cudaStream_t stream) {
  if (table_dtype == kF32)
    return gather_out<float>(bias, out_dtype, table, pairs, npairs, rows, H, stream);
  if (table_dtype == kF16)
    return gather_out<__half>(bias, out_dtype, table, pairs, npairs, rows, H, stream);
  return gather_out<__nv_bfloat16>(bias, out_dtype, table, pairs, npairs, rows, H, stream);
}

int launch_relative_position_bias_grad(const BiasGradArgs& a, cudaStream_t stream) {
  if (a.grad_dtype == kF32) return grad_out<float>(a, stream);
  if (a.grad_dtype == kF16) return grad_out<__half>(a, stream);
  return grad_out<__nv_bfloat16>(a, stream);
}

}  // namespace crumpet
