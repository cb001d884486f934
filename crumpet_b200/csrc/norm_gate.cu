// crumpet_b200: the passes between two branches of a block, forward and backward.
//
//   n      = post_norm(branch), or branch                (LayerNorm over the C channels)
//   out    = residual + s[sample] * gate * n             (drop path scale, layer scale; each 1
//                                                         where not given), rounded to its type
//   normed = pre_norm(out)                               (the next branch's LayerNorm)
//
// and, from the gradients of out and normed (t is the gradient of the sum):
//   t       = grad_out + LN'(grad_normed)                -> grad of residual
//   u       = s t,  grad_gate = sum_rows u n,  v = gate u
//   LN'(v)                                               -> grad of branch
// with LN'(g) = rstd (g w - mean(g w) - x^ mean(g w x^)), and the column sums of g x^ and g for
// the norms' weights and biases.  Mean and rstd are taken again from the rows at hand (they are
// in registers anyway), in fp32 with two passes, so nothing is kept but out and branch.
//
// HBM traffic bounds both: every row is read once and written once.  A row belongs to P lanes
// of 8 channels each (P a power of two, from one lane to sixteen warps); a lane's 8 channels
// neighbour each other (16-byte accesses) where C and the pointers allow, else lie P apart.
// Column sums stay in registers over all rows of a lane, are joined per CTA and written as one
// partial row per CTA, which a second kernel adds up in a fixed order: no atomics.
//
// Measured: forward of 110592 x 48 in bf16 12 us, 6.6 us of HBM time; backward of 442368 x 48, fp16
// branch and fp32 stream, all sums, 102 us, 59 us of HBM time: the shuffles of the rows' sums keep
// the load/store pipe 69 % busy and 128 registers hold it to 16 warps per SM.  A ring of
// asynchronous copies in shared memory instead of the registers' row ahead took 120 us.
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

constexpr int kMaxLanes = 512;  // C <= 4096
constexpr int kSums = 5;        // gate, post weight, post bias, pre weight, pre bias

struct Args {
  const void* branch;
  const void* residual;  // forward
  void* out;             // forward: written; backward: read
  void* normed;
  const void* grad_out;
  const void* grad_normed;
  void* grad_residual;
  void* grad_branch;
  float* partial;  // [kSums][CTAs][C]
  const float* gate;
  const float* row_scale;
  const float* post_w;
  const float* post_b;
  const float* pre_w;
  const float* pre_b;
  long long M;
  long long rows_per_sample;
  DivMod32 by_sample;  // by rows_per_sample, for rows that fit 32 bits
  int C, P;
  float eps, inv_c;
};

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

// The 8 channels of a lane: [8 lane, 8 lane + 8) (VEC), or lane + k P.
template <bool VEC>
struct Lane {
  int lane, P, C;
  __device__ __forceinline__ int col(int k) const { return VEC ? 8 * lane + k : lane + k * P; }
  __device__ __forceinline__ bool has(int k) const { return VEC ? 8 * lane < C : col(k) < C; }

  // the lane's values of a row as they are stored (0 past the row or the last channel)
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, bool in, Pack8<T>& w) const {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < int(sizeof(w)) / 16; ++k)
        reinterpret_cast<uint4*>(&w)[k] =
            in && has(0) ? ldg_stream(reinterpret_cast<const uint4*>(row + 8 * lane) + k)
                         : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w.v[k] = in && has(k) ? row[col(k)] : from_f32<T>(0.f);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, bool in, const float (&x)[8]) const {
    if constexpr (VEC) {
      if (!in || !has(0)) return;
      Pack8<T> w;
#pragma unroll
      for (int k = 0; k < 8; ++k) w.v[k] = from_f32<T>(x[k]);
#pragma unroll
      for (int k = 0; k < int(sizeof(w)) / 16; ++k)
        stg(reinterpret_cast<uint4*>(row + 8 * lane) + k, reinterpret_cast<const uint4*>(&w)[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (in && has(k)) row[col(k)] = from_f32<T>(x[k]);
    }
  }
  // fp32 parameters of the lane's channels (0 past the last); from L1 after the first row
  __device__ __forceinline__ void param(const float* p, float (&x)[8]) const {
    if constexpr (VEC) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
      if (has(0)) {
        a = __ldg(reinterpret_cast<const float4*>(p + 8 * lane));
        b = __ldg(reinterpret_cast<const float4*>(p + 8 * lane) + 1);
      }
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = has(k) ? __ldg(p + col(k)) : 0.f;
    }
  }
};

template <typename T>
__device__ __forceinline__ void unpack(const Pack8<T>& w, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = to_f32(w.v[k]);
}

// The row's factor: 1, or its sample's.
__device__ __forceinline__ float row_factor(const Args& a, long long row, bool in) {
  if (a.row_scale == nullptr || !in) return 1.f;
  return __ldg(a.row_scale + (a.M <= 0xffffffffLL ? (long long)a.by_sample.div(uint32_t(row))
                                                  : row / a.rows_per_sample));
}

// Sums of two values over the P lanes of a row.  BLOCK: the row spans warps of the CTA, whose
// parts meet in shared memory (every thread of the CTA takes part).
template <bool BLOCK>
__device__ __forceinline__ float2 row_sum(float a, float b, int P, float2* sh) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    if (!BLOCK && o >= P) break;
    a += __shfl_xor_sync(~0u, a, o);
    b += __shfl_xor_sync(~0u, b, o);
  }
  if constexpr (BLOCK) {
    const int warp = threadIdx.x >> 5, first = warp / (P >> 5) * (P >> 5);
    __syncthreads();  // the previous sum's parts have been read
    if ((threadIdx.x & 31) == 0) sh[warp] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
    for (int w = 0; w < (P >> 5); ++w) {
      a += sh[first + w].x;
      b += sh[first + w].y;
    }
  }
  return make_float2(a, b);
}

// x -> x^ = (x - mean) rstd, 0 in the lane's channels past C, for one or two rows' values whose
// sums go together; the rstds.  Two passes: the variance is of the centred values.
template <bool VEC, bool BLOCK, bool TWO>
__device__ __forceinline__ float2 normalise(float (&x)[8], float (&y)[8], const Lane<VEC>& ln,
                                            const Args& a, float2* sh) {
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    s += x[k];
    if constexpr (TWO) t += y[k];
  }
  const float2 mean = row_sum<BLOCK>(s, t, a.P, sh);
  s = t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[k] = ln.has(k) ? fmaf(-mean.x, a.inv_c, x[k]) : 0.f;
    s = fmaf(x[k], x[k], s);
    if constexpr (TWO) {
      y[k] = ln.has(k) ? fmaf(-mean.y, a.inv_c, y[k]) : 0.f;
      t = fmaf(y[k], y[k], t);
    }
  }
  const float2 var = row_sum<BLOCK>(s, t, a.P, sh);
  const float2 rstd = make_float2(1.f / sqrtf(fmaf(var.x, a.inv_c, a.eps)),
                                  TWO ? 1.f / sqrtf(fmaf(var.y, a.inv_c, a.eps)) : 0.f);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    x[k] *= rstd.x;
    if constexpr (TWO) y[k] *= rstd.y;
  }
  return rstd;
}

// Both kernels fetch a row ahead: its loads are in flight through the sums and shuffles of the
// row before.
template <typename T, typename R, bool VEC, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kMaxLanes : 256) norm_gate_forward_kernel(const Args a) {
  __shared__ float2 sh[16];
  const int per_cta = blockDim.x / a.P;
  const Lane<VEC> ln{int(threadIdx.x) % a.P, a.P, a.C};
  const long long step = (long long)gridDim.x * per_cta;
  long long row = blockIdx.x * (long long)per_cta + threadIdx.x / a.P;
  Pack8<T> yp;
  Pack8<R> rp;
  ln.fetch(static_cast<const T*>(a.branch) + row * a.C, row < a.M, yp);
  ln.fetch(static_cast<const R*>(a.residual) + row * a.C, row < a.M, rp);
  for (long long r0 = blockIdx.x * (long long)per_cta; r0 < a.M; r0 += step, row += step) {
    const bool in = row < a.M;
    float y[8], r[8], w[8], b[8];
    unpack(yp, y);
    unpack(rp, r);
    if (r0 + step < a.M) {
      ln.fetch(static_cast<const T*>(a.branch) + (row + step) * a.C, row + step < a.M, yp);
      ln.fetch(static_cast<const R*>(a.residual) + (row + step) * a.C, row + step < a.M, rp);
    }
    const float s = row_factor(a, row, in);
    if (a.post_w) {
      normalise<VEC, BLOCK, false>(y, y, ln, a, sh);
      ln.param(a.post_w, w);
      ln.param(a.post_b, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = fmaf(y[k], w[k], b[k]);
    }
    if (a.gate) {
      ln.param(a.gate, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] *= w[k];
    }
    // rounded once, and the next norm reads what is stored
#pragma unroll
    for (int k = 0; k < 8; ++k) r[k] = to_f32(from_f32<R>(fmaf(y[k], s, r[k])));
    ln.store(static_cast<R*>(a.out) + row * a.C, in, r);
    if (a.pre_w) {
      normalise<VEC, BLOCK, false>(r, r, ln, a, sh);
      ln.param(a.pre_w, w);
      ln.param(a.pre_b, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = fmaf(r[k], w[k], b[k]);
      ln.store(static_cast<T*>(a.normed) + row * a.C, in, r);
    }
  }
}

// What a lane reads of a row backward
template <typename T, typename R, bool VEC>
struct BackRow {
  Pack8<R> t, x;  // grad_out, out
  Pack8<T> g, y;  // grad_normed, branch
  __device__ __forceinline__ void fetch(const Args& a, const Lane<VEC>& ln, long long row,
                                        bool need_branch) {
    const bool in = row < a.M;
    const long long at = row * a.C;
    ln.fetch(static_cast<const R*>(a.grad_out) + at, in, t);
    if (a.pre_w) {
      ln.fetch(static_cast<const R*>(a.out) + at, in, x);
      ln.fetch(static_cast<const T*>(a.grad_normed) + at, in, g);
    }
    if (need_branch) ln.fetch(static_cast<const T*>(a.branch) + at, in, y);
  }
};

template <typename T, typename R, bool VEC, bool BLOCK, bool POST>
__global__ void __launch_bounds__(BLOCK ? kMaxLanes : 256, BLOCK ? 1 : 2)
norm_gate_backward_kernel(const Args a) {
  __shared__ float2 sh[16];
  __shared__ float cols[kMaxLanes * 8];
  const int per_cta = blockDim.x / a.P;
  const Lane<VEC> ln{int(threadIdx.x) % a.P, a.P, a.C};
  const bool need_branch = POST || a.gate != nullptr;
  const long long step = (long long)gridDim.x * per_cta;
  long long row = blockIdx.x * (long long)per_cta + threadIdx.x / a.P;
  float sum[kSums][8] = {};
  BackRow<T, R, VEC> ahead;
  ahead.fetch(a, ln, row, need_branch);
  for (long long r0 = blockIdx.x * (long long)per_cta; r0 < a.M; r0 += step, row += step) {
    const bool in = row < a.M;
    float t[8], x[8], g[8], y[8], w[8];
    unpack(ahead.t, t);
    if (a.pre_w) {
      unpack(ahead.x, x);
      unpack(ahead.g, g);
    }
    if (need_branch) unpack(ahead.y, y);
    if (r0 + step < a.M) ahead.fetch(a, ln, row + step, need_branch);
    const float s = row_factor(a, row, in);
    float2 rstd = make_float2(0.f, 0.f);  // of out and of branch
    if constexpr (POST) {
      if (a.pre_w) {
        rstd = normalise<VEC, BLOCK, true>(x, y, ln, a, sh);
      } else {
        rstd.y = normalise<VEC, BLOCK, false>(y, y, ln, a, sh).x;
      }
    } else if (a.pre_w) {
      rstd = normalise<VEC, BLOCK, false>(x, x, ln, a, sh);
    }
    if (a.pre_w) {
      ln.param(a.pre_w, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum[3][k] = fmaf(g[k], x[k], sum[3][k]);
        sum[4][k] += g[k];
        g[k] *= w[k];
        s1 += g[k];
        s2 = fmaf(g[k], x[k], s2);
      }
      const float2 m = row_sum<BLOCK>(s1, s2, a.P, sh);
      const float m1 = m.x * a.inv_c, m2 = m.y * a.inv_c;
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = fmaf(g[k] - m1 - x[k] * m2, rstd.x, t[k]);
    }
    ln.store(static_cast<R*>(a.grad_residual) + row * a.C, in, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] *= s;
    if (a.gate) {
      float q[8];
      if constexpr (POST) {
        ln.param(a.post_w, w);
        ln.param(a.post_b, q);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[0][k] = fmaf(t[k], fmaf(y[k], w[k], q[k]), sum[0][k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[0][k] = fmaf(t[k], y[k], sum[0][k]);
      }
      ln.param(a.gate, q);
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] *= q[k];
    }
    if constexpr (POST) {
      ln.param(a.post_w, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum[1][k] = fmaf(t[k], y[k], sum[1][k]);
        sum[2][k] += t[k];
        t[k] *= w[k];
        s1 += t[k];
        s2 = fmaf(t[k], y[k], s2);
      }
      const float2 m = row_sum<BLOCK>(s1, s2, a.P, sh);
      const float m1 = m.x * a.inv_c, m2 = m.y * a.inv_c;
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = (t[k] - m1 - y[k] * m2) * rstd.y;
    }
    ln.store(static_cast<T*>(a.grad_branch) + row * a.C, in, t);
  }

  // the CTA's column sums: over the rows of a warp by shuffles, over the warps in shared memory
  const int slots = a.P < 32 ? blockDim.x / 32 : blockDim.x / a.P;  // parts of every column
  const int slot = a.P < 32 ? threadIdx.x / 32 : threadIdx.x / a.P;
  const bool writes = a.P >= 32 || (threadIdx.x & 31) < a.P;
  for (int q = 0; q < kSums; ++q) {
    if (q == 0 ? !a.gate : q < 3 ? !POST : !a.pre_w) continue;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // a chain of selects: no dynamic index into the register array
      v[k] = q == 0 ? sum[0][k] : q == 1 ? sum[1][k] : q == 2 ? sum[2][k] : q == 3 ? sum[3][k]
                                                                                  : sum[4][k];
      for (int o = a.P; o < 32; o <<= 1) v[k] += __shfl_xor_sync(~0u, v[k], o);
    }
    __syncthreads();
    if (writes) {
#pragma unroll
      for (int k = 0; k < 8; ++k) cols[slot * a.P * 8 + ln.col(k)] = v[k];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
      float s = 0.f;
      for (int p = 0; p < slots; ++p) s += cols[p * a.P * 8 + c];
      a.partial[((long long)q * gridDim.x + blockIdx.x) * a.C + c] = s;
    }
  }
}

struct Sums {
  float* to[kSums];
};

// 32 columns of one of the sums per CTA: 32 rows of partials at a time
__global__ void __launch_bounds__(1024) norm_gate_columns_kernel(Sums out, const float* partial,
                                                                 int ctas, int C) {
  __shared__ float part[32][33];
  const int q = blockIdx.y, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float* to = out.to[q];
  if (to == nullptr) return;  // the whole CTA
  const int c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < C)
#pragma unroll 8
    for (int r = ty; r < ctas; r += 32) s += partial[((long long)q * ctas + r) * C + c];
  part[ty][tx] = s;
  __syncthreads();
  float v = part[tx][ty];  // column ty of the 32, its 32 parts across the warp
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if (tx == 0 && blockIdx.x * 32 + ty < C) to[blockIdx.x * 32 + ty] = v;
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int lanes_for(int64_t C) {
  int p = 1;
  while (int64_t(p) * 8 < C) p *= 2;
  return p;
}

int threads_for(int lanes) { return lanes > 256 ? lanes : 256; }

int64_t backward_ctas(int64_t M, int64_t C) {
  const int lanes = lanes_for(C), threads = threads_for(lanes);
  const int64_t tiles = (M + threads / lanes - 1) / (threads / lanes);
  const int64_t most = int64_t(sm_count()) * (threads > 256 ? 1 : 2);
  return tiles < most ? tiles : most;
}

Args make_args(const NormGateArgs& n) {
  Args a{};
  a.branch = n.branch;
  a.residual = n.residual;
  a.out = n.out;
  a.normed = n.normed;
  a.grad_out = n.grad_out;
  a.grad_normed = n.grad_normed;
  a.grad_residual = n.grad_residual;
  a.grad_branch = n.grad_branch;
  a.partial = n.partial;
  a.gate = n.gate;
  a.row_scale = n.row_scale;
  a.post_w = n.post_w;
  a.post_b = n.post_b;
  a.pre_w = n.pre_w;
  a.pre_b = n.pre_b;
  a.M = n.M;
  a.rows_per_sample = n.samples > 0 ? n.M / n.samples : 1;
  if (a.rows_per_sample <= 0xffffffffLL) a.by_sample = DivMod32::make(uint32_t(a.rows_per_sample));
  a.C = int(n.C);
  a.P = lanes_for(n.C);
  a.eps = n.eps;
  a.inv_c = 1.f / float(n.C);
  return a;
}

template <typename T, typename R>
int forward(const NormGateArgs& n, cudaStream_t stream) {
  const Args a = make_args(n);
  const int threads = threads_for(a.P);
  const int64_t tiles = (a.M + threads / a.P - 1) / (threads / a.P);
  const int64_t most = int64_t(sm_count()) * 8;
  const unsigned grid = unsigned(tiles < most ? tiles : most);
  const bool vec = a.C % 8 == 0 && aligned16(a.branch) && aligned16(a.residual) &&
                   aligned16(a.out) && aligned16(a.normed) && aligned16(a.gate) &&
                   aligned16(a.post_w) && aligned16(a.post_b) && aligned16(a.pre_w) &&
                   aligned16(a.pre_b);
  if (a.P > 32) {
    if (vec) norm_gate_forward_kernel<T, R, true, true><<<grid, threads, 0, stream>>>(a);
    else norm_gate_forward_kernel<T, R, false, true><<<grid, threads, 0, stream>>>(a);
  } else {
    if (vec) norm_gate_forward_kernel<T, R, true, false><<<grid, threads, 0, stream>>>(a);
    else norm_gate_forward_kernel<T, R, false, false><<<grid, threads, 0, stream>>>(a);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "norm gate residual launch");
}

template <typename T, typename R, bool POST>
void backward_rows(const Args& a, unsigned grid, int threads, bool vec, cudaStream_t stream) {
  if (a.P > 32) {
    if (vec) norm_gate_backward_kernel<T, R, true, true, POST><<<grid, threads, 0, stream>>>(a);
    else norm_gate_backward_kernel<T, R, false, true, POST><<<grid, threads, 0, stream>>>(a);
  } else {
    if (vec) norm_gate_backward_kernel<T, R, true, false, POST><<<grid, threads, 0, stream>>>(a);
    else norm_gate_backward_kernel<T, R, false, false, POST><<<grid, threads, 0, stream>>>(a);
  }
}

template <typename T, typename R>
int backward(const NormGateArgs& n, cudaStream_t stream) {
  const Args a = make_args(n);
  const int threads = threads_for(a.P);
  const unsigned grid = unsigned(backward_ctas(n.M, n.C));
  const bool vec = a.C % 8 == 0 && aligned16(a.branch) && aligned16(a.out) &&
                   aligned16(a.grad_out) && aligned16(a.grad_normed) &&
                   aligned16(a.grad_residual) && aligned16(a.grad_branch) && aligned16(a.gate) &&
                   aligned16(a.post_w) && aligned16(a.post_b) && aligned16(a.pre_w);
  if (a.post_w) backward_rows<T, R, true>(a, grid, threads, vec, stream);
  else backward_rows<T, R, false>(a, grid, threads, vec, stream);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "norm gate residual backward launch");
  if (a.gate || a.post_w || a.pre_w) {
    const Sums s{{a.gate ? n.grad_gate : nullptr, a.post_w ? n.grad_post_w : nullptr,
                  a.post_w ? n.grad_post_b : nullptr, a.pre_w ? n.grad_pre_w : nullptr,
                  a.pre_w ? n.grad_pre_b : nullptr}};
    norm_gate_columns_kernel<<<dim3(unsigned((a.C + 31) / 32), kSums), 1024, 0, stream>>>(
        s, a.partial, int(grid), a.C);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "norm gate residual columns launch");
  }
  return kOk;
}

}  // namespace

int64_t norm_gate_backward_partials(int64_t M, int64_t C) {
  if (M < 1 || C < 1 || C > 8 * kMaxLanes) return 0;
  return backward_ctas(M, C) * kSums * C;
}

int launch_norm_gate(const NormGateArgs& n, cudaStream_t stream) {
  if (n.dtype == kF32) return forward<float, float>(n, stream);
  if (n.dtype == kF16)
    return n.stream_dtype == kF32 ? forward<__half, float>(n, stream)
                                  : forward<__half, __half>(n, stream);
  return n.stream_dtype == kF32 ? forward<__nv_bfloat16, float>(n, stream)
                                : forward<__nv_bfloat16, __nv_bfloat16>(n, stream);
}

int launch_norm_gate_backward(const NormGateArgs& n, cudaStream_t stream) {
  if (n.dtype == kF32) return backward<float, float>(n, stream);
  if (n.dtype == kF16)
    return n.stream_dtype == kF32 ? backward<__half, float>(n, stream)
                                  : backward<__half, __half>(n, stream);
  return n.stream_dtype == kF32 ? backward<__nv_bfloat16, float>(n, stream)
                                : backward<__nv_bfloat16, __nv_bfloat16>(n, stream);
}

}  // namespace crumpet
