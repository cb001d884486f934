// crumpet_b200: learned relative-position bias by buckets, and its gradient.
//
//   bias[h, i, j] = table[pairs[i, j], h]
//   grad_table[t, h] = sum over the pairs (i, j) of bucket t of grad[h, i, j]
//
// Both move one value per (head, pair) and compute next to nothing, so memory traffic and, at
// a Swin window's size (343 x 343 pairs), launch latency bound them.
//
// Forward: a thread takes one pair (two neighbouring ones where the output's type has 16 bits,
// so its stores have 4 bytes) and a 16-byte vector of heads, which lie next to each other in the
// table: one gather per 4 or 8 heads, and every store of a warp is contiguous.
//
// Gradient: no atomics, so the sum's order never changes.  The caller sorted the pairs by
// bucket once (`order`) and cut every bucket into items of a bounded number of pairs; one
// warp sums an item in a fixed order, in fp32, for kUnit heads at a time: a pair's place is read
// once for all of them and the gathers, which are all latency, go out together.  The warps of a CTA
// take neighbouring items, whose pairs are neighbours in memory, so the sectors that one gather
// opens serve the others from L1.  Buckets of several items are finished by a second kernel.
//
// Pairs and the plan's entries are checked against their tensors (device error word, bit 2): a
// comparison per pair beside its gathers, which changed neither time below by more than 0.7 us.
//
// Measured: 24 heads of a 7 x 7 x 7 window in fp32 (no bucket of several items): 5 us forward and 14 us
// gradient, 25 MB that would take 3.8 us; 1024 x 1024 pairs in logarithmic buckets, 16 heads, bf16:
// 7 us forward, 17 and 4 us gradient, 12 us of them HBM time.  The gradient's gathers (84 % of the
// warps resident, nearly all waiting for loads) are the larger part.  Eight heads per warp were
// slower than four.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 4;   // heads that a warp gathers together
constexpr int kJoinThreads = 1024;
constexpr int kGradThreads = 512;  // 16 neighbouring items per CTA share the sectors in L1

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

// V heads (16 bytes of the table, or one) of PP neighbouring pairs per thread
template <typename T, typename O, int V, int PP>
__global__ void __launch_bounds__(kThreads)
bias_gather_kernel(O* bias, const T* table, unsigned rows, const int* pairs, long long npairs,
                   int H, int* error) {
  struct alignas(V * sizeof(T)) Heads {
    T v[V];
  };
  struct alignas(PP * sizeof(O)) Out {
    O v[PP];
  };
  struct alignas(PP * 4) Pairs {
    int v[PP];
  };
  const long long i = (blockIdx.x * (long long)kThreads + threadIdx.x) * PP;
  if (i >= npairs) return;
  const int h = blockIdx.y * V;
  const Pairs at = *reinterpret_cast<const Pairs*>(pairs + i);
  Heads w[PP];
  unsigned most = 0;
#pragma unroll
  for (int u = 0; u < PP; ++u) {
    most = max(most, unsigned(at.v[u]));
    w[u] = *reinterpret_cast<const Heads*>(
        table + (long long)min(unsigned(at.v[u]), rows - 1) * H + h);
  }
  if (most >= rows) {  // a bucket outside the table: no bias
    atomicOr(error, 2);
#pragma unroll
    for (int u = 0; u < PP; ++u)
      if (unsigned(at.v[u]) >= rows) w[u] = Heads{};
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    Out o;
#pragma unroll
    for (int u = 0; u < PP; ++u) o.v[u] = from_float<O>(to_float(w[u].v[k]));
    *reinterpret_cast<Out*>(bias + (h + k) * npairs + i) = o;
  }
}

struct GradBuckets {
  const int* order;      // [npairs] pairs sorted by bucket
  const int* items;      // [n_items][3]: bucket, begin, end (into order)
  const int* multi;      // [n_multi][3]: bucket, first item, last item + 1
  long long n_items, n_multi, npairs, rows;  // rows of the table
  int H;
  int* error;  // what points outside its tensor is flagged here and left out
};

// One warp per item and kUnit heads.  An item whose bucket is whole writes the table's gradient,
// the others their part: partial[item, h].
template <typename G, typename O>
__global__ void __launch_bounds__(kGradThreads, 4)
bias_grad_kernel(O* grad_table, float* partial, const G* grad, GradBuckets b) {
  const int lane = threadIdx.x & 31;
  const long long item = blockIdx.x * (long long)(kGradThreads / 32) + (threadIdx.x >> 5);
  if (item >= b.n_items) return;
  const int h = blockIdx.y * kUnit;
  const int bucket = b.items[3 * item], begin = b.items[3 * item + 1], end = b.items[3 * item + 2];
  if (bucket >= b.rows || (bucket < 0 && partial == nullptr) || begin < 0 || end > b.npairs) {
    atomicOr(b.error, 2);
    return;  // the whole warp
  }
  const int units = min(kUnit, b.H - h);
  const G* src = grad + h * b.npairs;
  const unsigned npairs = unsigned(b.npairs);
  unsigned most = 0;
  float sum[kUnit] = {};
  // n rounds of 32 pairs, all their places read at once (counted unsigned: they run past `end`,
  // which may be the last int)
  auto rounds = [&](auto n_tag, unsigned e0) {
    constexpr int n = decltype(n_tag)::value;
    unsigned at[n];
#pragma unroll
    for (int r = 0; r < n; ++r) {
      const bool in = e0 + 32 * r < unsigned(end);
      at[r] = in ? unsigned(__ldg(b.order + e0 + 32 * r)) : ~0u;
      most = max(most, in ? at[r] : 0u);
    }
#pragma unroll
    for (int u = 0; u < kUnit; ++u) {
      if (u >= units) break;
#pragma unroll
      for (int r = 0; r < n; ++r)
        if (at[r] < npairs) sum[u] += to_float(__ldg(src + u * b.npairs + at[r]));
    }
  };
  unsigned e = begin;
  for (; int(end - e) > 64; e += 128) rounds(std::integral_constant<int, 4>{}, e + lane);
  if (int(end - e) > 32) rounds(std::integral_constant<int, 2>{}, e + lane);
  else if (int(end - e) > 0) rounds(std::integral_constant<int, 1>{}, e + lane);
  if (most >= npairs && end > begin) atomicOr(b.error, 2);
#pragma unroll
  for (int u = 0; u < kUnit; ++u) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[u] += __shfl_xor_sync(~0u, sum[u], o);
    if (lane == u && u < units) {
      if (bucket >= 0) grad_table[(long long)bucket * b.H + h + u] = from_float<O>(sum[u]);
      else partial[item * b.H + h + u] = sum[u];
    }
  }
}

// One CTA per bucket of several items and 32 heads: a lane per head, the items dealt to the warps.
template <typename O>
__global__ void __launch_bounds__(kJoinThreads)
bias_grad_join_kernel(O* grad_table, const float* partial, GradBuckets b) {
  __shared__ float part[kJoinThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long k = blockIdx.x;
  const int h = blockIdx.y * 32 + lane;
  const int bucket = b.multi[3 * k], first = b.multi[3 * k + 1], last = b.multi[3 * k + 2];
  if (bucket < 0 || bucket >= b.rows || first < 0 || last > b.n_items) {
    if (threadIdx.x == 0) atomicOr(b.error, 2);
    return;  // the whole CTA
  }
  float sum = 0.f;
  if (h < b.H) {
#pragma unroll 8
    for (unsigned i = first + warp; i < unsigned(last); i += kJoinThreads / 32)
      sum += __ldg(partial + (long long)i * b.H + h);
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || h >= b.H) return;
#pragma unroll
  for (int w = 1; w < kJoinThreads / 32; ++w) sum += part[w][lane];
  grad_table[(long long)bucket * b.H + h] = from_float<O>(sum);
}

template <typename T, typename O, int V, int PP>
void gather(void* bias, const void* table, int64_t rows, const int* pairs, int64_t npairs, int64_t H,
            int* error, cudaStream_t stream) {
  const int64_t per = int64_t(kThreads) * PP;
  bias_gather_kernel<T, O, V, PP><<<dim3(unsigned((npairs + per - 1) / per), unsigned(H / V)),
                                    kThreads, 0, stream>>>(
      static_cast<O*>(bias), static_cast<const T*>(table), unsigned(rows), pairs, npairs, int(H),
      error);
}

template <typename T, typename O>
int launch_gather(void* bias, const void* table, int64_t rows, const int* pairs, int64_t npairs,
                  int64_t H, cudaStream_t stream) {
  int* error = nullptr;
  if (int e = training_error_word(&error)) return e;
  constexpr int V = 16 / sizeof(T), PP = 4 / sizeof(O);
  const auto aligned = [](const void* p, uintptr_t n) {
    return reinterpret_cast<uintptr_t>(p) % n == 0;
  };
  const bool heads = H % V == 0 && aligned(table, 16);
  const bool two = npairs % PP == 0 && aligned(bias, 4) && aligned(pairs, 4 * PP);
  if (heads && two) gather<T, O, V, PP>(bias, table, rows, pairs, npairs, H, error, stream);
  else if (heads) gather<T, O, V, 1>(bias, table, rows, pairs, npairs, H, error, stream);
  else if (two) gather<T, O, 1, PP>(bias, table, rows, pairs, npairs, H, error, stream);
  else gather<T, O, 1, 1>(bias, table, rows, pairs, npairs, H, error, stream);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "relative position bias launch");
}

template <typename T>
int gather_out(void* bias, int out_dtype, const void* table, int64_t rows, const int* pairs,
               int64_t npairs, int64_t H, cudaStream_t stream) {
  if (out_dtype == kF32)
    return launch_gather<T, float>(bias, table, rows, pairs, npairs, H, stream);
  if (out_dtype == kF16)
    return launch_gather<T, __half>(bias, table, rows, pairs, npairs, H, stream);
  return launch_gather<T, __nv_bfloat16>(bias, table, rows, pairs, npairs, H, stream);
}

template <typename G, typename O>
int launch_grad(const BiasGradArgs& a, cudaStream_t stream) {
  GradBuckets b{a.order, a.items, a.multi, a.n_items, a.n_multi, a.npairs, a.table_rows, int(a.H),
                nullptr};
  if (int e = training_error_word(&b.error)) return e;
  constexpr int items = kGradThreads / 32;
  bias_grad_kernel<G, O><<<dim3(unsigned((a.n_items + items - 1) / items),
                                unsigned((a.H + kUnit - 1) / kUnit)),
                           kGradThreads, 0, stream>>>(static_cast<O*>(a.grad_table), a.partial,
                                                      static_cast<const G*>(a.grad), b);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "relative position bias gradient launch");
  if (a.n_multi > 0) {
    bias_grad_join_kernel<O><<<dim3(unsigned(a.n_multi), unsigned((a.H + 31) / 32)), kJoinThreads,
                               0, stream>>>(static_cast<O*>(a.grad_table), a.partial, b);
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
                                  int64_t table_rows, const int* pairs, int64_t npairs, int64_t H,
                                  cudaStream_t stream) {
  if (table_dtype == kF32)
    return gather_out<float>(bias, out_dtype, table, table_rows, pairs, npairs, H, stream);
  if (table_dtype == kF16)
    return gather_out<__half>(bias, out_dtype, table, table_rows, pairs, npairs, H, stream);
  return gather_out<__nv_bfloat16>(bias, out_dtype, table, table_rows, pairs, npairs, H, stream);
}

int launch_relative_position_bias_grad(const BiasGradArgs& a, cudaStream_t stream) {
  if (a.grad_dtype == kF32) return grad_out<float>(a, stream);
  if (a.grad_dtype == kF16) return grad_out<__half>(a, stream);
  return grad_out<__nv_bfloat16>(a, stream);
}

}  // namespace crumpet
