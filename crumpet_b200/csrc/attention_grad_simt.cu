// crumpet_b200: window attention for training on the inputs that neither attention_grad.cu nor
// attention_grad_tf32.cu takes: head dims 64 to 256, and in 16 bits windows of more than 352
// tokens or unaligned tensors.
//
// The formulas of attention_grad.cu in plain fp32 arithmetic.  Tiles of 32 tokens of the other
// side stream through shared memory (as fp32):
//   * forward: one query row per lane group, online softmax (no gradient; the training forward of
//              the same inputs);
//   * rows:    one query row per lane group; a first sweep over the keys takes the row's
//              statistics with an online softmax (maximum, sum, sum of p dp), a second dq;
//   * columns: one key row per lane group, one sweep over the queries for dk and dv;
//   * bias:    one 32 x 32 tile of (query, key) pairs of one head per CTA, summed over the
//              windows of its share in registers.
// A row belongs to 4 lanes that share out the other side's tokens (head dims up to 32: each lane
// keeps the row's channels in registers, so a product is free of shuffles, and four times the
// threads hide the latency of small batches), or to D / 32 lanes of 32 channels each, whose
// partial products are added with shuffles.  The bias (+ mask) of the CTA's rows is gathered
// into shared memory once where it fits.
//
// Bound by: 11 products of depth D per score, three of them the repeated scores, fed from shared
// memory, where a 16-byte load gives four multiply-adds per lane.  At 64 windows of 125 tokens,
// three heads of 16 channels, as fp32: 28 us forward, 48 us rows, 49 us columns, 33 us bias; the
// loads from shared memory take 62 % and 69 % of their rate in the first two, FMA 20 %.  Two rows
// per lane halve those loads but need twice the registers, and came out level (33, 50 us); a tile
// loaded ahead into registers, too (28, 51, 49 us).  At 16 windows of 216 tokens, three heads of
// 64 channels, fp32: 68 us forward, 127 us rows, 96 us columns, 92 us bias.  (16-bit tensors are
// multiplied in fp32 here too, at the same rate.)
#include <cmath>

#include "attention_grad_f32.cuh"
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

using namespace grad_f32;

constexpr int kThreads = 128;
constexpr int kTile = 32;  // tokens streamed at a time
constexpr int kBiasBytes = 64 * 1024;  // most shared memory for the bias of a CTA's rows
template <int D>
struct Shape {
  static constexpr int KL = D <= 32 ? 4 : 1;            // lanes that share out the tokens
  static constexpr int TPR = D <= 32 ? 1 : D / 32;      // lanes that share out the channels
  static constexpr int LANES = KL * TPR;                // lanes per row
  static constexpr int E = D / TPR;                     // channels per lane
  static constexpr int R = kThreads / LANES;            // rows per CTA
  static constexpr int SLICE = E + 4;  // slices (of a row, or of the KL rows read at once) in
                                       // different banks
  static constexpr int ROW = TPR * SLICE;
  static constexpr int STAGED = 2 * kTile * ROW * 4 + kTile * 8;  // bytes of a tile and statistics
  // most of any call: the bias, and a byte per row and per token that it holds
  static constexpr int MOST = STAGED + kBiasBytes + R + kBiasBytes / (4 * R) + kTile;
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
// sums over the lanes that share out the tokens
template <typename S>
__device__ __forceinline__ float over_tokens(float v) {
#pragma unroll
  for (int o = 1; o < S::KL; o <<= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
template <typename S>
__device__ __forceinline__ void over_tokens(float (&a)[S::E]) {
#pragma unroll
  for (int e = 0; e < S::E; ++e) a[e] = over_tokens<S>(a[e]);
}

// kTile token rows starting at j0 (zero past N) as fp32 into pitched shared memory
template <typename T, int D>
__device__ __forceinline__ void stage(const Params& p, float* dst, const T* src, long long stride,
                                      int j0) {
  using S = Shape<D>;
#pragma unroll 4
  for (int f = threadIdx.x; f < kTile * (D / 4); f += kThreads) {
    const int j = f / (D / 4), d = f % (D / 4) * 4;
    *reinterpret_cast<float4*>(dst + j * S::ROW + (d / S::E) * S::SLICE + d % S::E) =
        j0 + j < p.N ? load4(p, src + (j0 + j) * stride + d) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// At 16 channels registers are held to six CTAs per SM (five for the columns, which keep two
// sums per lane): 38 against 48 us forward and 57 against 71 us for the rows at 64 windows of 125
// tokens and three heads, where the gathers' latency counts.  A limit at the wider shapes spills.
template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kThreads, D == 16 && MODE != kCols ? 6 : D == 16 ? 5 : 1) grad_simt_kernel(const Params p) {
  using S = Shape<D>;
  constexpr bool COLS = MODE == kCols;
  extern __shared__ float4 smem4[];
  float* xs = reinterpret_cast<float*>(smem4);       // K (or Q) rows
  float* ys = xs + kTile * S::ROW;                   // V (or dO) rows
  float2* stat = reinterpret_cast<float2*>(ys + kTile * S::ROW);
  float* tile = reinterpret_cast<float*>(stat + kTile);  // bias + mask [row][pitch]
  const int tid = threadIdx.x, row = tid / S::LANES;
  const int part = tid % S::TPR, first = tid % S::KL;  // channel slice, first token of a tile
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

  // this row's own vectors: q and do (rows), k and v (columns)
  float a0[S::E], a1[S::E];
  auto own = [&](float (&x)[S::E], const T* at) {
#pragma unroll
    for (int e = 0; e < S::E; e += 4) {
      const float4 w = valid ? load4(p, at + part * S::E + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[e] = w.x, x[e + 1] = w.y, x[e + 2] = w.z, x[e + 3] = w.w;
    }
  };
  own(a0, (COLS ? k : q) + i * tok);
  if constexpr (MODE == kRows) own(a1, g + i * hd);
  if constexpr (COLS) own(a1, v + i * tok);
  const float c1 = p.scale * kLog2e;
  // the bias (+ mask) of `cols` tokens from j0 on, for the CTA's rows: lanes along the keys, which
  // neighbour in `pairs`, eight gathers in flight per thread
  const int whole = p.bias_pitch;  // the pitch of all of it in shared memory, or 0: tile by tile
  const int pitch = whole ? whole : kTile + 1;
  const int warp = tid / 32, lane = tid % 32;
  // roll-side codes of the CTA's rows and of the gathered tokens (windows at a seam only)
  uint8_t* row_code = reinterpret_cast<uint8_t*>(tile + S::R * pitch);
  uint8_t* tok_code = row_code + S::R;
  auto gather = [&](int j0, int cols) {
    if (last != 0) {
      for (int f = tid; f < S::R + cols; f += kThreads) {
        const int t = f < S::R ? r0 + f : j0 + f - S::R;
        row_code[f] = t < p.N ? uint8_t(side_code(p, t)) : uint8_t(0);
      }
      __syncthreads();  // `last` is the CTA's
    }
    // eight pairs at a time: their indices, then their table entries, so that both loads of eight
    // are in flight (with clamped indices; what lies past the end is replaced afterwards)
    constexpr int WARPS = kThreads / 32, BATCH = 8;
    unsigned most = 0;
    const int across = COLS ? S::R : cols, along = COLS ? cols : S::R;
    for (int x = lane; x < across; x += 32) {
      for (int y0 = warp; y0 < along; y0 += WARPS * BATCH) {
        unsigned bucket[BATCH];
        float v[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int y = y0 + u * WARPS;
          const int gi = min(r0 + (COLS ? x : y), p.N - 1), gj = min(j0 + (COLS ? y : x), p.N - 1);
          bucket[u] = bucket_of(p, (long long)(COLS ? gj : gi) * p.N + (COLS ? gi : gj), most);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) v[u] = bias_of<T>(p, h, bucket[u]);
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int y = y0 + u * WARPS;
          if (y >= along) continue;
          const int r = COLS ? x : y, j = COLS ? y : x;
          if (last != 0 && ((row_code[r] ^ tok_code[j]) & last)) v[u] += -100.f * kLog2e;
          // past the end of the softmax a pair drops out; past the rows nothing is stored
          tile[r * pitch + j] = j0 + j >= p.N ? -INFINITY : v[u];
        }
      }
    }
    check_buckets(p, most);
  };
  if (whole) gather(0, (p.N + kTile - 1) / kTile * kTile);
  auto fetch = [&](int j0) {
    __syncthreads();  // the previous tile is no longer read
    stage<T, D>(p, xs, COLS ? q : k, tok, j0);
    stage<T, D>(p, ys, COLS ? g : v, COLS ? hd : tok, j0);
    if (!whole) gather(j0, kTile);
    if (COLS && tid < kTile) stat[tid] = j0 + tid < p.N ? stats[j0 + tid] : make_float2(0.f, 0.f);
    __syncthreads();
    return tile + row * pitch + (whole ? j0 : 0);
  };

  if constexpr (!COLS) {
    // per lane: maximum, sum of exponentials, and the sum of p dp or (forward) of p v
    float m = -1e30f, l = 0.f, dp = 0.f;
    float acc[S::E] = {};
    for (int j0 = 0; j0 < p.N; j0 += kTile) {
      const float* bias = fetch(j0);
      float s[kTile / S::KL], mc = m;
#pragma unroll
      for (int n = 0; n < kTile / S::KL; ++n) {
        const int j = first + n * S::KL;
        s[n] = fmaf(dot<S>(a0, xs + j * S::ROW + part * S::SLICE), c1, bias[j]);
        mc = fmaxf(mc, s[n]);
      }
      const float alpha = exp2f(m - mc);
      l *= alpha;
      dp *= alpha;
      if constexpr (MODE == kForward) {
#pragma unroll
        for (int e = 0; e < S::E; ++e) acc[e] *= alpha;
      }
      m = mc;
#pragma unroll
      for (int n = 0; n < kTile / S::KL; ++n) {
        const float* yr = ys + (first + n * S::KL) * S::ROW + part * S::SLICE;
        const float e = exp2f(s[n] - m);
        l += e;
        if constexpr (MODE == kForward) add<S>(acc, e, yr);
        else dp = fmaf(e, dot<S>(a1, yr), dp);
      }
    }
    float top = m;
#pragma unroll
    for (int o = 1; o < S::KL; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float f = exp2f(m - top);
    l = over_tokens<S>(l * f);
    if constexpr (MODE == kForward) {
#pragma unroll
      for (int e = 0; e < S::E; ++e) acc[e] *= f;
      over_tokens<S>(acc);
      if (!valid || first != 0) return;
      T* out = static_cast<T*>(p.out) + ((long long)b * p.N + i) * hd + h * D + part * S::E;
      const float inv = 1.f / l;
#pragma unroll
      for (int e = 0; e < S::E; ++e) out[e] = store_as<T>(acc[e] * inv);
    } else {
      dp = over_tokens<S>(dp * f);
      const float lse = top + log2f(l), delta = dp / l;
      if (valid && part == 0 && first == 0) stats[i] = make_float2(lse, delta);
      for (int j0 = 0; j0 < p.N; j0 += kTile) {
        const float* bias = fetch(j0);
#pragma unroll 4
        for (int n = 0; n < kTile / S::KL; ++n) {
          const int j = first + n * S::KL;
          const float* xr = xs + j * S::ROW + part * S::SLICE;
          const float e = exp2f(fmaf(dot<S>(a0, xr), c1, bias[j]) - lse);
          add<S>(acc, e * (dot<S>(a1, ys + j * S::ROW + part * S::SLICE) - delta), xr);
        }
      }
      over_tokens<S>(acc);
      if (!valid || first != 0) return;
      T* out = static_cast<T*>(p.dqkv) + ((long long)b * p.N + i) * tok + h * D + part * S::E;
#pragma unroll
      for (int e = 0; e < S::E; ++e) out[e] = store_as<T>(acc[e] * p.scale);
    }
  } else {
    float dk[S::E] = {}, dv[S::E] = {};
    for (int j0 = 0; j0 < p.N; j0 += kTile) {
      const float* bias = fetch(j0);
#pragma unroll 4
      for (int n = 0; n < kTile / S::KL; ++n) {
        const int j = first + n * S::KL;
        const float* xr = xs + j * S::ROW + part * S::SLICE;
        const float* yr = ys + j * S::ROW + part * S::SLICE;
        const float2 st = stat[j];
        const float e = exp2f(fmaf(dot<S>(a0, xr), c1, bias[j]) - st.x);
        const float ds = e * (dot<S>(a1, yr) - st.y);
        add<S>(dv, e, yr);
        add<S>(dk, ds, xr);
      }
    }
    over_tokens<S>(dk);
    over_tokens<S>(dv);
    if (!valid || first != 0) return;
    T* out = static_cast<T*>(p.dqkv) + ((long long)b * p.N + i) * tok + hd + h * D + part * S::E;
#pragma unroll
    for (int e = 0; e < S::E; ++e) {
      out[e] = store_as<T>(dk[e] * p.scale);
      out[hd + e] = store_as<T>(dv[e]);
    }
  }
}

// dbias of one 32 x 32 tile of pairs of one head, over the windows of one share.  A thread keeps
// one key and 8 queries; CH channels at a time, the key's in registers, the queries' read from
// shared memory by all threads at once.
template <typename T, int CH>
__global__ void __launch_bounds__(kThreads, CH == 16 ? 6 : 1) grad_bias_simt_kernel(const Params p, int D) {
  __shared__ __align__(16) float qs[kTile * CH], gs[kTile * CH];
  const int tiles = (p.N + kTile - 1) / kTile;
  long long blk = blockIdx.x;
  const int share = int(blk % p.S);
  blk /= p.S;
  const int jt = int(blk % tiles);
  blk /= tiles;
  const int it = int(blk % tiles), h = int(blk / tiles);
  const int j = jt * kTile + threadIdx.x % kTile;
  const int ib = threadIdx.x / kTile * 8;  // this thread's 8 query rows
  const long long hd = (long long)p.H * D, tok = 3 * hd;
  const float c1 = p.scale * kLog2e;
  float base[8], sum[8];
  uint32_t apart[8];
  unsigned most = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = it * kTile + ib + u;
    const bool in = i < p.N && j < p.N;
    base[u] = in ? bias_of<T>(p, h, bucket_of(p, (long long)i * p.N + j, most)) : 0.f;
    apart[u] = in && p.analytic ? side_code(p, i) ^ side_code(p, j) : 0u;
    sum[u] = 0.f;
  }
  check_buckets(p, most);
  for (int b = share; b < p.B; b += p.S) {
    const T* q = static_cast<const T*>(p.qkv) + (long long)b * p.N * tok + h * D;
    const T* g = static_cast<const T*>(p.dout) + (long long)b * p.N * hd + h * D;
    float s[8] = {}, d[8] = {};
    for (int c0 = 0; c0 < D; c0 += CH) {
      float kr[CH], vr[CH];
      const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < CH; c += 4) {
        const float4 x = j < p.N ? load4(p, q + j * tok + hd + c0 + c) : z;
        const float4 y = j < p.N ? load4(p, q + j * tok + 2 * hd + c0 + c) : z;
        kr[c] = x.x, kr[c + 1] = x.y, kr[c + 2] = x.z, kr[c + 3] = x.w;
        vr[c] = y.x, vr[c + 1] = y.y, vr[c + 2] = y.z, vr[c + 3] = y.w;
      }
      __syncthreads();
#pragma unroll 2
      for (int f = threadIdx.x; f < kTile * CH / 4; f += kThreads) {
        const int i = it * kTile + f / (CH / 4), c = c0 + f % (CH / 4) * 4;
        reinterpret_cast<float4*>(qs)[f] = i < p.N ? load4(p, q + i * tok + c) : z;
        reinterpret_cast<float4*>(gs)[f] = i < p.N ? load4(p, g + i * hd + c) : z;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float4* qr = reinterpret_cast<const float4*>(qs + (ib + u) * CH);
        const float4* gr = reinterpret_cast<const float4*>(gs + (ib + u) * CH);
#pragma unroll
        for (int e = 0; e < CH / 4; ++e) {
          const float4 x = qr[e], y = gr[e];
          s[u] = fmaf(x.x, kr[4 * e], s[u]);
          d[u] = fmaf(y.x, vr[4 * e], d[u]);
          s[u] = fmaf(x.y, kr[4 * e + 1], s[u]);
          d[u] = fmaf(y.y, vr[4 * e + 1], d[u]);
          s[u] = fmaf(x.z, kr[4 * e + 2], s[u]);
          d[u] = fmaf(y.z, vr[4 * e + 2], d[u]);
          s[u] = fmaf(x.w, kr[4 * e + 3], s[u]);
          d[u] = fmaf(y.w, vr[4 * e + 3], d[u]);
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
      if (apart[u] & last) x += -100.f * kLog2e;
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

template <typename T, int D, int MODE>
int start(long long blocks, int smem, const Params& p, cudaStream_t stream) {
  const auto kernel = grad_simt_kernel<T, D, MODE>;
  static std::atomic<bool> allowed[64];  // per device
  if (int e = allow_smem(kernel, Shape<D>::MOST, allowed)) return e;
  kernel<<<unsigned(blocks), kThreads, smem, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention (simt) launch");
}

template <typename T, int D>
int launch(Params p, bool forward, cudaStream_t stream) {
  using S = Shape<D>;
  p.QB = (p.N + S::R - 1) / S::R;
  const long long blocks = (long long)p.B * p.H * p.QB;
  const long long tiles = (p.N + kTile - 1) / kTile;
  const long long bias_blocks = tiles * tiles * p.H * p.S;
  if (blocks > 0x7fffffffLL || bias_blocks > 0x7fffffffLL)
    return set_error(kErrInvalid, "too many windows x heads for one launch");
  // an odd pitch: lanes of neighbouring rows read different banks
  const int pitch = int(tiles) * kTile + 1;
  p.bias_pitch = S::R * pitch * 4 <= kBiasBytes ? pitch : 0;
  const int smem = S::STAGED + S::R * (p.bias_pitch ? pitch : kTile + 1) * 4 + S::R +
                   (p.bias_pitch ? int(tiles) * kTile : kTile);
  if (forward) return start<T, D, kForward>(blocks, smem, p, stream);
  if (int e = start<T, D, kRows>(blocks, smem, p, stream)) return e;
  if (int e = start<T, D, kCols>(blocks, smem, p, stream)) return e;
  constexpr int CH = D < 32 ? D : 32;
  grad_bias_simt_kernel<T, CH><<<unsigned(bias_blocks), kThreads, 0, stream>>>(p, D);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention gradient (simt) launch");
}

template <typename T>
int dispatch(const Params& p, int head_dim, bool forward, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {  // fp32 at these head dims: attention_grad_tf32.cu
    if (head_dim == 16) return launch<T, 16>(p, forward, stream);
    if (head_dim == 32) return launch<T, 32>(p, forward, stream);
  }
  switch (head_dim) {
    case 64: return launch<T, 64>(p, forward, stream);
    case 128: return launch<T, 128>(p, forward, stream);
    default: return launch<T, 256>(p, forward, stream);
  }
}

int launch_any(const AttnGradArgs& a, void* out, bool forward, cudaStream_t stream) {
  Params p{};
  p.qkv = a.qkv;
  p.dout = a.grad_out;
  p.dqkv = a.grad_qkv;
  p.dbias = a.grad_bias;
  p.stats = reinterpret_cast<float2*>(a.stats);
  p.out = out;
  p.table = a.table;
  p.pairs = a.pairs;
  p.table_f32 = a.table_f32 ? 1 : 0;
  p.table_rows = int(a.table_rows);
  if (int e = training_error_word(&p.error)) return e;
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
  p.vec = ((reinterpret_cast<uintptr_t>(a.qkv) | reinterpret_cast<uintptr_t>(a.grad_out) |
            reinterpret_cast<uintptr_t>(a.grad_qkv) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
  if (attention_tf32(a.dtype, a.head_dim))
    return launch_attention_tf32(p, int(a.head_dim), forward, stream);
  if (a.dtype == kF32) return dispatch<float>(p, int(a.head_dim), forward, stream);
  if (a.dtype == kF16) return dispatch<__half>(p, int(a.head_dim), forward, stream);
  return dispatch<__nv_bfloat16>(p, int(a.head_dim), forward, stream);
}

}  // namespace

// Shares of the windows for the bias kernel: enough CTAs for the GPU's SMs, eight per SM.
int64_t attention_grad_shares_simt(int64_t B, int64_t H, int64_t N, int64_t head_dim, int dtype) {
  if (attention_tf32(dtype, head_dim)) return attention_grad_shares_tf32(B, H, N);
  const int64_t tiles = (N + kTile - 1) / kTile;
  const int64_t s = 148 * 8 / (tiles * tiles * H);
  return s < 1 ? 1 : s > B ? (B > 0 ? B : 1) : s > 16 ? 16 : s;
}

int launch_attention_grad_simt(const AttnGradArgs& a, cudaStream_t stream) {
  return launch_any(a, nullptr, false, stream);
}

int launch_attention_train_simt(const AttnGradArgs& a, void* out, cudaStream_t stream) {
  return launch_any(a, out, true, stream);
}

}  // namespace crumpet
