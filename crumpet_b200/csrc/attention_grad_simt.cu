// crumpet_b200: gradient of the window attention for the inputs attention_grad.cu does not
// take: float32 qkv, head dims 64 to 256, windows of more than 352 tokens, unaligned tensors.
//
// The formulas of attention_grad.cu in plain fp32 arithmetic, in three kernels that stream
// tiles of the other side through shared memory (fp32, 32 tokens at a time):
//   * rows:    one query row per lane group; a first sweep over the keys takes the row's
//              statistics with an online softmax (maximum, sum, sum of p dp), a second dq;
//   * columns: one key row per lane group, one sweep over the queries for dk and dv;
//   * bias:    one 32 x 32 tile of (query, key) pairs of one head per CTA, summed over the
//              windows of its share in registers.
// A row belongs to TPR = max(1, D / 32) neighbouring lanes of E = D / TPR channels, whose
// partial products are added with shuffles.  fp32 FMA work bounds it: 11 products of depth D
// per score, three of them the repeated scores.
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

constexpr int kThreads = 128;
constexpr int kTile = 32;  // tokens streamed at a time
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void* qkv;    // [B, N, 3, H, D]
  const void* dout;   // [B, N, H, D]
  void* dqkv;         // [B, N, 3, H, D]
  float* dbias;       // [S, H, N, N]
  float2* stats;      // [B, H, N]
  const void* table;  // [T, H]
  const int* pairs;   // [N, N]
  int table_f32, analytic;
  int nwd, nwh, nww, wsd, wsh, wsw, ssd, ssh, ssw;
  int B, H, N, QB, S;
  float scale;
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

// bias (+ mask) of one pair times log2 e
template <typename T>
__device__ __forceinline__ float extra(const Params& p, int h, int i, int j, uint32_t last) {
  const long long t = p.pairs[(long long)i * p.N + j];
  float v = p.table_f32 ? __ldg(static_cast<const float*>(p.table) + t * p.H + h)
                        : load(static_cast<const T*>(p.table), t * p.H + h);
  if (last != 0 && ((side_code(p, i) ^ side_code(p, j)) & last)) v += -100.f;
  return v * kLog2e;
}

template <int D>
struct Shape {
  static constexpr int TPR = D >= 64 ? D / 32 : 1;
  static constexpr int E = D / TPR;
  static constexpr int R = kThreads / TPR;            // rows per CTA
  static constexpr int SLICE = E + (TPR > 1 ? 4 : 0);  // slices of a row in different banks
  static constexpr int ROW = TPR * SLICE;
  static constexpr int PAD = kTile + 1;
  static constexpr int SMEM = (2 * kTile * ROW + R * PAD) * 4 + kTile * 8;
  static_assert(E % 4 == 0 && E <= 32, "channels per lane");
};

template <typename S>
__device__ __forceinline__ float dot(const float (&a)[S::E], const float* row) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < S::E / 4; ++e) {
    const float4 v = reinterpret_cast<const float4*>(row)[e];
    s = fmaf(a[4 * e], v.x, s);
    s = fmaf(a[4 * e + 1], v.y, s);
    s = fmaf(a[4 * e + 2], v.z, s);
    s = fmaf(a[4 * e + 3], v.w, s);
  }
#pragma unroll
  for (int o = 1; o < S::TPR; o <<= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}
template <typename S>
__device__ __forceinline__ void add(float (&a)[S::E], float w, const float* row) {
#pragma unroll
  for (int e = 0; e < S::E / 4; ++e) {
    const float4 v = reinterpret_cast<const float4*>(row)[e];
    a[4 * e] = fmaf(w, v.x, a[4 * e]);
    a[4 * e + 1] = fmaf(w, v.y, a[4 * e + 1]);
    a[4 * e + 2] = fmaf(w, v.z, a[4 * e + 2]);
    a[4 * e + 3] = fmaf(w, v.w, a[4 * e + 3]);
  }
}

// kTile token rows starting at j0 (zero past N) as fp32 into pitched shared memory
template <typename T, int D>
__device__ __forceinline__ void stage(float* dst, const T* src, long long stride, int j0, int N) {
  using S = Shape<D>;
  for (int f = threadIdx.x; f < kTile * D; f += kThreads) {
    const int j = f / D, d = f % D;
    dst[j * S::ROW + (d / S::E) * S::SLICE + d % S::E] =
        j0 + j < N ? load(src, (long long)(j0 + j) * stride + d) : 0.f;
  }
}

template <typename T, int D, bool COLS>
__global__ void __launch_bounds__(kThreads) grad_simt_kernel(const Params p) {
  using S = Shape<D>;
  extern __shared__ float4 smem4[];
  float* xs = reinterpret_cast<float*>(smem4);       // K (or Q) rows
  float* ys = xs + kTile * S::ROW;                   // V (or dO) rows
  float* tile = ys + kTile * S::ROW;                 // bias + mask of rows x streamed tokens
  float2* stat = reinterpret_cast<float2*>(tile + S::R * S::PAD + ((S::R * S::PAD) & 1));
  const int tid = threadIdx.x, row = tid / S::TPR, part = tid % S::TPR;
  long long blk = blockIdx.x;
  const int qb = int(blk % p.QB);
  blk /= p.QB;
  const int h = int(blk % p.H), b = int(blk / p.H);
  const int r0 = qb * S::R, i = r0 + row;
  const bool valid = i < p.N;
  const uint32_t last = last_axes(p, b);
  const long long hd = (long long)p.H * D, tok = 3 * hd;
  const T* q = static_cast<const T*>(p.qkv) + (long long)b * p.N * tok + h * D;
  const T* k = q + hd;
  const T* v = k + hd;
  const T* g = static_cast<const T*>(p.dout) + (long long)b * p.N * hd + h * D;
  float2* stats = p.stats + ((long long)b * p.H + h) * p.N;

  // this row's own two vectors: q and do (rows), k and v (columns)
  float a0[S::E], a1[S::E];
#pragma unroll
  for (int e = 0; e < S::E; ++e) {
    const long long d = part * S::E + e;
    a0[e] = valid ? load(COLS ? k : q, i * tok + d) : 0.f;
    a1[e] = !valid ? 0.f : COLS ? load(v, i * tok + d) : load(g, i * hd + d);
  }
  const float c1 = p.scale * kLog2e;
  auto fetch = [&](int j0) {
    __syncthreads();  // the previous tile is no longer read
    stage<T, D>(xs, COLS ? q : k, tok, j0, p.N);
    stage<T, D>(ys, COLS ? g : v, COLS ? hd : tok, j0, p.N);
    for (int f = tid; f < S::R * kTile; f += kThreads) {
      // along the keys, which neighbour in `pairs`
      const int r = COLS ? f % S::R : f / kTile, j = COLS ? f / S::R : f % kTile;
      const int gi = r0 + r, gj = j0 + j;
      float x = -INFINITY;  // past the end: drops out of the softmax
      if (gj < p.N) x = gi < p.N ? extra<T>(p, h, COLS ? gj : gi, COLS ? gi : gj, last) : 0.f;
      tile[r * S::PAD + j] = x;
    }
    if (COLS && tid < kTile) stat[tid] = j0 + tid < p.N ? stats[j0 + tid] : make_float2(0.f, 0.f);
    __syncthreads();
  };

  if constexpr (!COLS) {
    float m = -INFINITY, l = 0.f, dp = 0.f;
    for (int j0 = 0; j0 < p.N; j0 += kTile) {
      fetch(j0);
      float s[kTile], mc = m;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        s[j] = fmaf(dot<S>(a0, xs + j * S::ROW + part * S::SLICE), c1, tile[row * S::PAD + j]);
        mc = fmaxf(mc, s[j]);
      }
      const float alpha = exp2f(m - mc);  // the first tile: 2^-inf = 0
      l *= alpha;
      dp *= alpha;
      m = mc;
#pragma unroll
      for (int j = 0; j < kTile; ++j) {
        const float e = exp2f(s[j] - m);
        l += e;
        dp = fmaf(e, dot<S>(a1, ys + j * S::ROW + part * S::SLICE), dp);
      }
    }
    const float lse = m + log2f(l), delta = dp / l;
    if (valid && part == 0) stats[i] = make_float2(lse, delta);
    float acc[S::E] = {};
    for (int j0 = 0; j0 < p.N; j0 += kTile) {
      fetch(j0);
#pragma unroll 4
      for (int j = 0; j < kTile; ++j) {
        const float* xr = xs + j * S::ROW + part * S::SLICE;
        const float e = exp2f(fmaf(dot<S>(a0, xr), c1, tile[row * S::PAD + j]) - lse);
        add<S>(acc, e * (dot<S>(a1, ys + j * S::ROW + part * S::SLICE) - delta), xr);
      }
    }
    if (!valid) return;
    T* out = static_cast<T*>(p.dqkv) + ((long long)b * p.N + i) * tok + h * D + part * S::E;
#pragma unroll
    for (int e = 0; e < S::E; ++e) out[e] = store_as<T>(acc[e] * p.scale);
  } else {
    float dk[S::E] = {}, dv[S::E] = {};
    for (int j0 = 0; j0 < p.N; j0 += kTile) {
      fetch(j0);
#pragma unroll 4
      for (int j = 0; j < kTile; ++j) {
        const float* xr = xs + j * S::ROW + part * S::SLICE;
        const float* yr = ys + j * S::ROW + part * S::SLICE;
        const float2 st = stat[j];
        const float e = exp2f(fmaf(dot<S>(a0, xr), c1, tile[row * S::PAD + j]) - st.x);
        const float ds = e * (dot<S>(a1, yr) - st.y);
        add<S>(dv, e, yr);
        add<S>(dk, ds, xr);
      }
    }
    if (!valid) return;
    T* out = static_cast<T*>(p.dqkv) + ((long long)b * p.N + i) * tok + hd + h * D + part * S::E;
#pragma unroll
    for (int e = 0; e < S::E; ++e) {
      out[e] = store_as<T>(dk[e] * p.scale);
      out[hd + e] = store_as<T>(dv[e]);
    }
  }
}

// dbias of one 32 x 32 tile of pairs of one head, over the windows of one share: a thread
// keeps 8 pairs.  Channels pass through shared memory 32 at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads) grad_bias_simt_kernel(const Params p, int D) {
  constexpr int CH = 32, P = CH + 1;
  __shared__ float qs[kTile * P], gs[kTile * P], ks[kTile * P], vs[kTile * P];
  const int tiles = (p.N + kTile - 1) / kTile;
  long long blk = blockIdx.x;
  const int share = int(blk % p.S);
  blk /= p.S;
  const int jt = int(blk % tiles);
  blk /= tiles;
  const int it = int(blk % tiles), h = int(blk / tiles);
  const int jj = threadIdx.x % kTile, j = jt * kTile + jj;
  const int ib = threadIdx.x / kTile * 8;  // this thread's 8 query rows
  const long long hd = (long long)p.H * D, tok = 3 * hd;
  const float c1 = p.scale * kLog2e;
  float base[8], apart[8], sum[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = it * kTile + ib + u;
    const bool in = i < p.N && j < p.N;
    base[u] = in ? extra<T>(p, h, i, j, 0u) : 0.f;
    apart[u] = in && p.analytic ? float(side_code(p, i) ^ side_code(p, j)) : 0.f;
    sum[u] = 0.f;
  }
  for (int b = share; b < p.B; b += p.S) {
    const T* q = static_cast<const T*>(p.qkv) + (long long)b * p.N * tok + h * D;
    const T* g = static_cast<const T*>(p.dout) + (long long)b * p.N * hd + h * D;
    float s[8] = {}, d[8] = {};
    for (int c0 = 0; c0 < D; c0 += CH) {
      const int w = min(CH, D - c0);
      __syncthreads();
      for (int f = threadIdx.x; f < kTile * CH; f += kThreads) {
        const int r = f / CH, c = f % CH;
        const int i = it * kTile + r, k = jt * kTile + r;
        qs[r * P + c] = i < p.N && c < w ? load(q, i * tok + c0 + c) : 0.f;
        gs[r * P + c] = i < p.N && c < w ? load(g, i * hd + c0 + c) : 0.f;
        ks[r * P + c] = k < p.N && c < w ? load(q, k * tok + hd + c0 + c) : 0.f;
        vs[r * P + c] = k < p.N && c < w ? load(q, k * tok + 2 * hd + c0 + c) : 0.f;
      }
      __syncthreads();
      for (int c = 0; c < w; ++c) {
        const float kk = ks[jj * P + c], vv = vs[jj * P + c];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          s[u] = fmaf(qs[(ib + u) * P + c], kk, s[u]);
          d[u] = fmaf(gs[(ib + u) * P + c], vv, d[u]);
        }
      }
    }
    const uint32_t last = last_axes(p, b);
    const float2* stats = p.stats + ((long long)b * p.H + h) * p.N;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = it * kTile + ib + u;
      if (i >= p.N || j >= p.N) continue;
      const float2 st = stats[i];
      float x = fmaf(s[u], c1, base[u]);
      if (uint32_t(apart[u]) & last) x += -100.f * kLog2e;
      sum[u] += exp2f(x - st.x) * (d[u] - st.y);
    }
  }
  float* out = p.dbias + ((long long)share * p.H + h) * p.N * p.N;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = it * kTile + ib + u;
    if (i < p.N && j < p.N) out[(long long)i * p.N + j] = sum[u];
  }
}

template <typename T, int D>
int launch(Params p, cudaStream_t stream) {
  using S = Shape<D>;
  p.QB = (p.N + S::R - 1) / S::R;
  const long long blocks = (long long)p.B * p.H * p.QB;
  const long long tiles = (p.N + kTile - 1) / kTile;
  const long long bias_blocks = tiles * tiles * p.H * p.S;
  if (blocks > 0x7fffffffLL || bias_blocks > 0x7fffffffLL)
    return set_error(kErrInvalid, "too many windows x heads for one launch");
  auto rows = grad_simt_kernel<T, D, false>;
  auto cols = grad_simt_kernel<T, D, true>;
  constexpr int smem = S::SMEM + 16;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(rows, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(cols, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return set_cuda_error(e, "attention gradient (simt) smem attribute");
  }
  rows<<<unsigned(blocks), kThreads, smem, stream>>>(p);
  cols<<<unsigned(blocks), kThreads, smem, stream>>>(p);
  grad_bias_simt_kernel<T><<<unsigned(bias_blocks), kThreads, 0, stream>>>(p, D);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention gradient (simt) launch");
}

template <typename T>
int dispatch(const Params& p, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 16: return launch<T, 16>(p, stream);
    case 32: return launch<T, 32>(p, stream);
    case 64: return launch<T, 64>(p, stream);
    case 128: return launch<T, 128>(p, stream);
    default: return launch<T, 256>(p, stream);
  }
}

}  // namespace

// Shares of the windows for the bias kernel: enough CTAs for the GPU's SMs, eight per SM.
int64_t attention_grad_shares_simt(int64_t B, int64_t H, int64_t N) {
  const int64_t tiles = (N + kTile - 1) / kTile;
  const int64_t s = 148 * 8 / (tiles * tiles * H);
  return s < 1 ? 1 : s > B ? (B > 0 ? B : 1) : s > 16 ? 16 : s;
}

int launch_attention_grad_simt(const AttnGradArgs& a, cudaStream_t stream) {
  Params p{};
  p.qkv = a.qkv;
  p.dout = a.grad_out;
  p.dqkv = a.grad_qkv;
  p.dbias = a.grad_bias;
  p.stats = reinterpret_cast<float2*>(a.stats);
  p.table = a.table;
  p.pairs = a.pairs;
  p.table_f32 = a.table_f32 ? 1 : 0;
  p.analytic = (a.shift[0] | a.shift[1] | a.shift[2]) != 0;
  p.nwd = int(a.nwin[0]);
  p.nwh = int(a.nwin[1]);
  p.nww = int(a.nwin[2]);
  p.wsd = int(a.win[0]);
  p.wsh = int(a.win[1]);
  p.wsw = int(a.win[2]);
  p.ssd = int(a.shift[0]);
  p.ssh = int(a.shift[1]);
  p.ssw = int(a.shift[2]);
  p.B = int(a.B);
  p.H = int(a.H);
  p.N = int(a.N);
  p.S = int(a.shares);
  p.scale = a.scale;
  if (a.dtype == kF32) return dispatch<float>(p, int(a.head_dim), stream);
  if (a.dtype == kF16) return dispatch<__half>(p, int(a.head_dim), stream);
  return dispatch<__nv_bfloat16>(p, int(a.head_dim), stream);
}

}  // namespace crumpet
