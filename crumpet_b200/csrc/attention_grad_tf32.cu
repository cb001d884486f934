// crumpet_b200: window attention for training in fp32 (head_dim 16 or 32), on the tensor cores.
//
// The formulas of attention_grad.cu.  A product of fp32 numbers is taken as three products of
// 11-bit (tf32) halves: x = hi + lo with hi = x cut to 11 bits and lo = x - hi (exact) cut
// likewise, and x y = hi hi + hi lo + lo hi; what is left out, lo lo (below 2^-20 of |x y|) and the
// bits cut from either lo (below 2^-21 each), is below 2^-19 and about 2^-22 on average, the size of
// an fp32 sum's own rounding.  The
// tensor core cuts its sums instead of rounding them, so sums over the tokens are kept in
// fragments for 32 tokens only and added to fp32 registers.  (An infinity comes out as NaN.)
//
// A warp takes 16 rows and streams the other side's tokens, which the CTA's four warps stage in
// shared memory 64 at a time; tiles of 16 x 8 scores stay in the fragment layout, in which the
// accumulators of one product are the operand of the next when the tokens of that product are
// counted as (2t, 2t + 1) instead of (t, t + 4).  In the same way a lane's channels are counted
// as four neighbours, so operands are read and results written 16 bytes at a time.
//   * forward: online softmax of the row, one sweep over the keys;
//   * rows:    a first sweep takes the row's maximum, sum and sum of p dp, a second dq;
//   * columns: the transposed scores, one sweep over the queries for dk and dv;
//   * bias:    a warp keeps 16 x 32 pairs of one head and sums ds over the windows of its share;
//              operands come straight from global memory, nothing is shared between warps.
//
// What bounds it: instructions, not the tensor cores (8.5 cycles per product and SM quarter when
// they are alone, 11 to 24 % busy here): splitting the staged operands, which every warp does for
// itself, and the softmax.  The bias kernel reads 6 KB per 16 x 32 pairs and window from L2 (3.4
// TB/s at 343 tokens).  At 64 windows of 125 tokens, three heads of 16 channels: forward 16 us,
// rows 26 us, columns 21 us, bias 25 us (fp32 arithmetic of attention_grad_simt.cu: 28, 48, 49,
// 33 us); of 343 tokens: 93, 181, 123 and 84 us, with 32 channels 156, 331, 193 and 113 us.
// Measured and not kept, at 125 tokens: two warps per 16 rows that share out the tokens (96 us in
// all, against 84 us before the third part was added to the sums' operands); tokens staged a tile
// ahead by asynchronous copies (94 us, the same, and 285 against 202 us at 144 tokens, where the
// second stage takes the place of the bias).
#include <cmath>
#include <type_traits>

#include "attention_grad_f32.cuh"
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

namespace {

using namespace grad_f32;

constexpr int kWarps = 4;            // most of a CTA
constexpr int kTile = 64;            // tokens staged at a time
constexpr int kBlock = 32;           // tokens whose scores a warp holds at a time
constexpr int kTiles = kBlock / 8;   // in tiles of 8

// 2^x by the hardware's approximation (2^-22 relative), which no range handling surrounds
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The two tf32 halves of x
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 rows of D channels as left operands: step s of 8 channels, hi and lo
template <int D>
struct Left {
  uint32_t hi[D / 8][4], lo[D / 8][4];
  // channels 4t to 4t + 3 of each 16 of rows g (u = 0) and g + 8 (u = 1)
  __device__ __forceinline__ void set(int u, int c, float4 v) {
    split(v.x, hi[2 * c][u], lo[2 * c][u]);
    split(v.y, hi[2 * c][u + 2], lo[2 * c][u + 2]);
    split(v.z, hi[2 * c + 1][u], lo[2 * c + 1][u]);
    split(v.w, hi[2 * c + 1][u + 2], lo[2 * c + 1][u + 2]);
  }
};
// s += left (16 rows) x 16 channels v (from 4t on) of 8 tokens, token g's at this lane
template <int D>
__device__ __forceinline__ void dot(float (&s)[4], const Left<D>& a, int c, float4 v) {
  uint32_t h[4], l[4];
  split(v.x, h[0], l[0]);
  split(v.y, h[1], l[1]);
  split(v.z, h[2], l[2]);
  split(v.w, h[3], l[3]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    mma(s, a.lo[2 * c + k], h[2 * k], h[2 * k + 1]);
    mma(s, a.hi[2 * c + k], l[2 * k], l[2 * k + 1]);
    mma(s, a.hi[2 * c + k], h[2 * k], h[2 * k + 1]);
  }
}
template <int D>
struct Stage {
  static constexpr int CTAS = D == 16 ? 4 : 2;  // per SM, that registers allow
  static constexpr int FLOATS = 2 * kTile * (D + 4) + 2 * kTile;  // x, y and statistics
  // bytes, most of any call: with the bias, and a byte per token of the longest window
  static constexpr int MOST = FLOATS * 4 + 64 * 1024 + 46400;
  static constexpr int ROW = D + 4;  // floats from a staged token to the next: both ways of
                                     // reading it (below) find the lanes' words in other banks
};
// s += left x the 8 staged tokens from `row` on (token g at this lane: row = its first)
template <int D>
__device__ __forceinline__ void dot_staged(float (&s)[4], const Left<D>& a, const float* rows,
                                           int g, int t) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
    dot<D>(s, a, c, *reinterpret_cast<const float4*>(rows + g * Stage<D>::ROW + 16 * c + 4 * t));
}
// acc += w (16 rows x 8 tokens, as the scores lie) x the 8 staged tokens' channels; acc[2c + k]
// holds channels 16c + 4t + k and 16c + 4t + 2 + k of rows g and g + 8
template <int D>
__device__ __forceinline__ void add_staged(float (&acc)[D / 8][4], const float (&w)[4],
                                           const float* rows, int g, int t) {
  uint32_t hi[4], lo[4];
  split(w[0], hi[0], lo[0]);
  split(w[2], hi[1], lo[1]);
  split(w[1], hi[2], lo[2]);
  split(w[3], hi[3], lo[3]);
  const float* at = rows + 2 * t * Stage<D>::ROW + 2 * g;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const float2 x = *reinterpret_cast<const float2*>(at + 16 * c);
    const float2 y = *reinterpret_cast<const float2*>(at + Stage<D>::ROW + 16 * c);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float xk = k ? x.y : x.x, yk = k ? y.y : y.x;
      uint32_t xh, xl, yh, yl;
      split(xk, xh, xl);
      split(yk, yh, yl);
      // what lo leaves of them: a weight of 1 gives the token's own value
      const float xr = xk - __uint_as_float(xh) - __uint_as_float(xl);
      const float yr = yk - __uint_as_float(yh) - __uint_as_float(yl);
      mma(acc[2 * c + k], hi, __float_as_uint(xr), __float_as_uint(yr));
      mma(acc[2 * c + k], lo, xh, yh);
      mma(acc[2 * c + k], hi, xl, yl);
      mma(acc[2 * c + k], hi, xh, yh);
    }
  }
}
template <int D>
__device__ __forceinline__ void join(float (&sum)[D / 8][4], const float (&part)[D / 8][4]) {
#pragma unroll
  for (int k = 0; k < D / 8; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[k][e] += part[k][e];
  }
}

// A CTA takes 16 rows per warp of one head and walks the windows of its share, so the bias of its
// rows, gathered once, stays in shared memory where it fits.
template <int D, int MODE>
__global__ void __launch_bounds__(32 * kWarps, Stage<D>::CTAS) grad_tf32_kernel(const Params p, int shares) {
  constexpr bool COLS = MODE == kCols;
  constexpr int ROW = Stage<D>::ROW;
  extern __shared__ float4 smem4[];
  float* xs = reinterpret_cast<float*>(smem4);                 // staged K (or Q)
  float* ys = xs + kTile * ROW;                                // staged V (or dO)
  float2* stat = reinterpret_cast<float2*>(ys + kTile * ROW);  // the staged queries' (columns)
  float* tile = xs + Stage<D>::FLOATS;                         // bias of the CTA's rows
  const int threads = blockDim.x, rows = threads / 2;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  int blk = blockIdx.x;
  const int qb = blk % p.QB;
  blk /= p.QB;
  const int h = blk % p.H, share = blk / p.H;
  const int r0 = qb * rows, i0 = r0 + warp * 16 + g;  // this lane's rows: i0 and i0 + 8
  const bool busy = r0 + warp * 16 < p.N;             // else the warp only helps staging
  const long long hd = (long long)p.H * D, tok = 3 * hd;
  const float c1 = p.scale * kLog2e;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);

  // The bias of the CTA's rows and `held` tokens: all of them, or tile by tile.  The rows' modes
  // keep it by rows; the columns', whose lanes gather along the rows (neighbours in `pairs`), by
  // tokens.  The pitches put the words that a warp reads at once into different banks.
  const bool whole = p.bias_pitch != 0;
  const int held = whole ? p.bias_pitch : kTile;
  const int pitch = COLS ? rows + 4 : held + 8;
  auto gather = [&](int j0) {
    // eight pairs at a time, so that their loads are in flight together (forward: the indices',
    // then the table's; the gradient finds the bias laid out where its own gradient will go)
    constexpr int BATCH = 8;
    unsigned most = 0;
    const int warps = threads / 32, across = COLS ? rows : held, along = COLS ? held : rows;
    for (int x = lane; x < across; x += 32) {
      for (int y0 = warp; y0 < along; y0 += warps * BATCH) {
        long long at[BATCH];
        float w[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int y = y0 + u * warps;
          const int gi = min(r0 + (COLS ? x : y), p.N - 1), gj = min(j0 + (COLS ? y : x), p.N - 1);
          at[u] = (long long)(COLS ? gj : gi) * p.N + (COLS ? gi : gj);
        }
        if constexpr (MODE == kForward) {
          unsigned bucket[BATCH];
#pragma unroll
          for (int u = 0; u < BATCH; ++u) bucket[u] = bucket_of(p, at[u], most);
#pragma unroll
          for (int u = 0; u < BATCH; ++u) w[u] = bias_of<float>(p, h, bucket[u]);
        } else {
          const float* dense = p.dbias + (long long)h * p.N * p.N;
#pragma unroll
          for (int u = 0; u < BATCH; ++u) w[u] = kLog2e * __ldg(dense + at[u]);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int y = y0 + u * warps;
          if (y >= along) continue;
          const int r = COLS ? x : y, j = COLS ? y : x;
          // past the last token a pair drops out; past the last row nothing is stored
          tile[COLS ? j * pitch + r : r * pitch + j] = j0 + j >= p.N ? -INFINITY : w[u];
        }
      }
    }
    if constexpr (MODE == kForward) check_buckets(p, most);
  };
  if (whole) gather(0);
  // roll-side codes: of this lane's rows, and of all tokens
  uint8_t* tok_code = reinterpret_cast<uint8_t*>(tile + (COLS ? held * pitch : rows * pitch));
  uint32_t row_code[2] = {};
  if (p.analytic) {
#pragma unroll
    for (int u = 0; u < 2; ++u) row_code[u] = i0 + 8 * u < p.N ? side_code(p, i0 + 8 * u) * 0x0101u : 0u;
    const int all = (p.N + kTile - 1) / kTile * kTile;
    for (int j = tid; j < all; j += threads)
      tok_code[j] = j < p.N ? uint8_t(side_code(p, j)) : uint8_t(0);
  }

  for (int b = share; b < p.B; b += shares) {
    const uint32_t last = last_axes(p, b);
    const float* q = static_cast<const float*>(p.qkv) + (long long)b * p.N * tok + h * D;
    const float* k = q + hd;
    const float* v = k + hd;
    const float* o = static_cast<const float*>(p.dout) + (long long)b * p.N * hd + h * D;
    float2* stats = p.stats + ((long long)b * p.H + h) * p.N;

    // the warp's own rows: q and do (rows), k and v (columns)
    Left<D> a0, a1;
    auto own = [&](Left<D>& x, const float* at, long long stride) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
          x.set(u, c,
                i0 + 8 * u < p.N ? load4(p, at + (i0 + 8 * u) * stride + 16 * c + 4 * t) : zero);
      }
    };
    own(a0, COLS ? k : q, tok);
    if constexpr (MODE == kRows) own(a1, o, hd);
    if constexpr (COLS) own(a1, v, tok);

    // stages tokens j0 on, zero past the last, as far as a warp reads them
    auto fetch = [&](int j0) {
      __syncthreads();  // the previous tile is no longer read
      const int count = min(kTile, (p.N - j0 + kBlock - 1) / kBlock * kBlock) * (D / 4);
      for (int f0 = tid; f0 < count; f0 += 2 * threads) {
        float4 x[2], y[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int f = f0 + u * threads, j = j0 + f / (D / 4), d = f % (D / 4) * 4;
          const bool in = f < count && j < p.N;
          x[u] = in ? load4(p, (COLS ? q : k) + j * tok + d) : zero;
          y[u] = in ? load4(p, COLS ? o + j * hd + d : v + j * tok + d) : zero;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int f = f0 + u * threads;
          if (f >= count) continue;
          float* at = xs + f / (D / 4) * ROW + f % (D / 4) * 4;
          *reinterpret_cast<float4*>(at) = x[u];
          *reinterpret_cast<float4*>(at + kTile * ROW) = y[u];
        }
      }
      if (!whole) gather(j0);
      if (COLS) {
        for (int j = tid; j < kTile; j += threads)
          stat[j] = j0 + j < p.N ? stats[j0 + j] : make_float2(0.f, 0.f);
      }
      __syncthreads();
    };
    // the staged tokens in blocks of four tiles of 8, or two where that is all there is
    auto each_block = [&](int j0, auto&& block) {
      for (int f = 0; f < kTile && j0 + f < p.N; f += kBlock) {
        if (p.N - j0 - f > kBlock / 2) block(std::integral_constant<int, kTiles>{}, f);
        else block(std::integral_constant<int, kTiles / 2>{}, f);
      }
    };
    // bias + mask of 8 tokens from staged token f on, as the scores lie
    auto bias_at = [&](float (&x)[4], int j0, int f) {
      const int at = (whole ? j0 : 0) + f + 2 * t;
      if constexpr (COLS) {
        const float* w = tile + at * pitch + warp * 16 + g;
        x[0] = w[0], x[1] = w[pitch], x[2] = w[8], x[3] = w[pitch + 8];
      } else {
        const float* w = tile + (warp * 16 + g) * pitch + at;
        const float2 u = *reinterpret_cast<const float2*>(w);
        const float2 u8 = *reinterpret_cast<const float2*>(w + 8 * pitch);
        x[0] = u.x, x[1] = u.y, x[2] = u8.x, x[3] = u8.y;
      }
      if (last != 0) {
        // two tokens' codes against each row's, copied beside itself
        const uint32_t two = *reinterpret_cast<const uint16_t*>(tok_code + j0 + f + 2 * t);
        const uint32_t sides = last * 0x0101u;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t apart = (two ^ row_code[u]) & sides;
          if (apart & 0xff) x[2 * u] += -100.f * kLog2e;
          if (apart & 0xff00) x[2 * u + 1] += -100.f * kLog2e;
        }
      }
    };
    // the sums' 4 channels from 16c + 4t on of row i0 + 8u, times its factor
    auto put = [&](const float (&x)[D / 8][4], float by, float by8, void* to, long long stride) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int i = i0 + 8 * u;
        if (i >= p.N) continue;
        const float f = u ? by8 : by;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float* at = static_cast<float*>(to) + i * stride + h * D + 16 * c + 4 * t;
          const float4 w = make_float4(x[2 * c][2 * u] * f, x[2 * c + 1][2 * u] * f,
                                       x[2 * c][2 * u + 1] * f, x[2 * c + 1][2 * u + 1] * f);
          if (p.vec) {
            *reinterpret_cast<float4*>(at) = w;
          } else {
            at[0] = w.x, at[1] = w.y, at[2] = w.z, at[3] = w.w;
          }
        }
      }
    };
    float* dqkv = static_cast<float*>(p.dqkv) + (long long)b * p.N * tok;

    if constexpr (!COLS) {
      // of rows i0 and i0 + 8: maximum, and this lane's part of the sums of exponentials and p dp
      float m[2] = {-1e30f, -1e30f}, l[2] = {}, dp[2] = {};
      float acc[D / 8][4] = {};
      for (int j0 = 0; j0 < p.N; j0 += kTile) {
        fetch(j0);
        if (!busy) continue;
        auto block = [&](auto tiles, int f) {
          constexpr int TILES = decltype(tiles)::value;
          float s[TILES][4], mc[2] = {m[0], m[1]};
#pragma unroll
          for (int n = 0; n < TILES; ++n) {
            float x[4], y[4] = {};
            bias_at(x, j0, f + 8 * n);
            dot_staged<D>(y, a0, xs + (f + 8 * n) * ROW, g, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[n][e] = fmaf(y[e], c1, x[e]);
              mc[e / 2] = fmaxf(mc[e / 2], s[n][e]);
            }
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            mc[u] = fmaxf(mc[u], __shfl_xor_sync(~0u, mc[u], 1));
            mc[u] = fmaxf(mc[u], __shfl_xor_sync(~0u, mc[u], 2));
            const float alpha = ex2(m[u] - mc[u]);
            m[u] = mc[u];
            l[u] *= alpha;
            dp[u] *= alpha;
            if constexpr (MODE == kForward) {
#pragma unroll
              for (int c = 0; c < D / 8; ++c) acc[c][2 * u] *= alpha, acc[c][2 * u + 1] *= alpha;
            }
          }
          [[maybe_unused]] float now[2][D / 8][4] = {};
#pragma unroll
          for (int n = 0; n < TILES; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[n][e] = ex2(s[n][e] - m[e / 2]);
              l[e / 2] += s[n][e];
            }
            const float* y = ys + (f + 8 * n) * ROW;
            if constexpr (MODE == kForward) {
              add_staged<D>(now[n % 2], s[n], y, g, t);
            } else {
              float d[4] = {};
              dot_staged<D>(d, a1, y, g, t);
#pragma unroll
              for (int e = 0; e < 4; ++e) dp[e / 2] = fmaf(s[n][e], d[e], dp[e / 2]);
            }
          }
          if constexpr (MODE == kForward) {
            join<D>(acc, now[0]);
            join<D>(acc, now[1]);
          }
        };
        each_block(j0, block);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          l[u] += __shfl_xor_sync(~0u, l[u], x);
          dp[u] += __shfl_xor_sync(~0u, dp[u], x);
        }
      }
      if constexpr (MODE == kForward) {
        put(acc, 1.f / l[0], 1.f / l[1], static_cast<float*>(p.out) + (long long)b * p.N * hd, hd);
      } else {
        const float lse[2] = {m[0] + log2f(l[0]), m[1] + log2f(l[1])};
        const float delta[2] = {dp[0] / l[0], dp[1] / l[1]};
        if (t < 2 && i0 + 8 * t < p.N)
          stats[i0 + 8 * t] = t ? make_float2(lse[1], delta[1]) : make_float2(lse[0], delta[0]);
        for (int j0 = 0; j0 < p.N; j0 += kTile) {
          if (p.N > kTile) fetch(j0);  // else all tokens are still there
          if (!busy) continue;
          auto block = [&](auto tiles, int f) {
            constexpr int TILES = decltype(tiles)::value;
            float now[2][D / 8][4] = {};
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
              float x[4], y[4] = {}, d[4] = {};
              bias_at(x, j0, f + 8 * n);
              dot_staged<D>(y, a0, xs + (f + 8 * n) * ROW, g, t);
              dot_staged<D>(d, a1, ys + (f + 8 * n) * ROW, g, t);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] = ex2(fmaf(y[e], c1, x[e]) - lse[e / 2]) * (d[e] - delta[e / 2]);
              add_staged<D>(now[n % 2], y, xs + (f + 8 * n) * ROW, g, t);
            }
            join<D>(acc, now[0]);
            join<D>(acc, now[1]);
          };
          each_block(j0, block);
        }
        put(acc, p.scale, p.scale, dqkv, tok);
      }
    } else {
      float dk[D / 8][4] = {}, dv[D / 8][4] = {};
      for (int j0 = 0; j0 < p.N; j0 += kTile) {
        fetch(j0);
        if (!busy) continue;
        auto block = [&](auto tiles, int f) {
          constexpr int TILES = decltype(tiles)::value;
          float pk[D / 8][4] = {}, pv[D / 8][4] = {};
#pragma unroll
          for (int n = 0; n < TILES; ++n) {
            float x[4], y[4] = {}, d[4] = {};
            bias_at(x, j0, f + 8 * n);
            const float4 st = *reinterpret_cast<const float4*>(stat + f + 8 * n + 2 * t);
            dot_staged<D>(y, a0, xs + (f + 8 * n) * ROW, g, t);
            dot_staged<D>(d, a1, ys + (f + 8 * n) * ROW, g, t);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              y[e] = ex2(fmaf(y[e], c1, x[e]) - (e % 2 ? st.z : st.x));
              d[e] = y[e] * (d[e] - (e % 2 ? st.w : st.y));
            }
            add_staged<D>(pv, y, ys + (f + 8 * n) * ROW, g, t);
            add_staged<D>(pk, d, xs + (f + 8 * n) * ROW, g, t);
          }
          join<D>(dk, pk);
          join<D>(dv, pv);
        };
        each_block(j0, block);
      }
      put(dk, p.scale, p.scale, dqkv + hd, tok);
      put(dv, 1.f, 1.f, dqkv + 2 * hd, tok);
    }
  }
}

// dbias of 16 queries x 32 keys of one head per warp, over the windows of one share
template <int D, bool VEC>
__global__ void __launch_bounds__(32 * kWarps) grad_bias_tf32_kernel(const Params p,
                                                                  long long warps) {
  const int lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  long long w = (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (w >= warps) return;
  const int jts = (p.N + kBlock - 1) / kBlock, its = (p.N + 15) / 16;
  const int jt = int(w % jts) * kBlock;
  w /= jts;
  const int i0 = int(w % its) * 16 + g;
  w /= its;
  const int share = int(w % p.S), h = int(w / p.S);
  const long long hd = (long long)p.H * D, tok = 3 * hd;
  const float c1 = p.scale * kLog2e;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  auto channels = [&](const float* at) {  // VEC: every tensor on 16-byte boundaries
    if constexpr (VEC) return __ldg(reinterpret_cast<const float4*>(at));
    else return make_float4(__ldg(at), __ldg(at + 1), __ldg(at + 2), __ldg(at + 3));
  };
  float base[kTiles][4], sum[kTiles][4] = {};
  uint32_t apart[kTiles];  // of each of four pairs, the axes on whose other side they lie: 4 x 8 bits
  {
    unsigned bucket[kTiles][4], most = 0;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bucket[n][e] = bucket_of(p, (long long)min(i0 + e / 2 * 8, p.N - 1) * p.N +
                                        min(jt + 8 * n + 2 * t + e % 2, p.N - 1), most);
    }
    check_buckets(p, most);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      apart[n] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        base[n][e] = bias_of<float>(p, h, bucket[n][e]);
        if (p.analytic)
          apart[n] |= (side_code(p, min(i0 + e / 2 * 8, p.N - 1)) ^
                       side_code(p, min(jt + 8 * n + 2 * t + e % 2, p.N - 1))) << (8 * e);
      }
    }
  }
  for (int b = share; b < p.B; b += p.S) {
    const float* q = static_cast<const float*>(p.qkv) + (long long)b * p.N * tok + h * D + 4 * t;
    const float* o = static_cast<const float*>(p.dout) + (long long)b * p.N * hd + h * D + 4 * t;
    const float2* stats = p.stats + ((long long)b * p.H + h) * p.N;
    const uint32_t last = last_axes(p, b) * 0x01010101u;
    // the loads of two tiles go out together, the first with those of the rows
    constexpr int AHEAD = kTiles / 2;
    float4 kv[AHEAD][2][D / 16];
    auto fetch = [&](int n0) {
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
        const int j = jt + 8 * (n0 + n) + g;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const float* at = q + j * tok + hd + 16 * c;
          kv[n][0][c] = j < p.N ? channels(at) : zero;
          kv[n][1][c] = j < p.N ? channels(at + hd) : zero;
        }
      }
    };
    float4 own[2][2][D / 16];
    float2 st[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = i0 + 8 * u;
      st[u] = i < p.N ? __ldg(stats + i) : make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        own[0][u][c] = i < p.N ? channels(q + i * tok + 16 * c) : zero;
        own[1][u][c] = i < p.N ? channels(o + i * hd + 16 * c) : zero;
      }
    }
    fetch(0);
    Left<D> a0, a1;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        a0.set(u, c, own[0][u][c]);
        a1.set(u, c, own[1][u][c]);
      }
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      if (n > 0 && n % AHEAD == 0) fetch(n);
      float s[4] = {}, d[4] = {};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        dot<D>(s, a0, c, kv[n % AHEAD][0][c]);
        dot<D>(d, a1, c, kv[n % AHEAD][1][c]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = fmaf(s[e], c1, base[n][e]);
        if (apart[n] & last & (0xffu << (8 * e))) x += -100.f * kLog2e;
        sum[n][e] += ex2(x - st[e / 2].x) * (d[e] - st[e / 2].y);
      }
    }
  }
  float* out = p.dbias + ((long long)share * p.H + h) * p.N * p.N;
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e / 2 * 8, j = jt + 8 * n + 2 * t + e % 2;
      if (i < p.N && j < p.N) out[(long long)i * p.N + j] = sum[n][e];
    }
  }
}

template <int D, int MODE>
int start(Params p, cudaStream_t stream) {
  if (p.B == 0) return kOk;
  const int warps = (p.N + 15) / 16 < kWarps ? (p.N + 15) / 16 : kWarps, rows = 16 * warps;
  p.QB = (p.N + rows - 1) / rows;
  // as many windows per CTA as leave the SMs one full round of CTAs
  const long long units = (long long)p.B * p.H * p.QB;
  const long long round = 148LL * Stage<D>::CTAS * kWarps / warps;
  const long long per = (units + round - 1) / round;
  const long long shares = (p.B + per - 1) / per, blocks = shares * p.H * p.QB;
  if (blocks > 0x7fffffffLL)
    return set_error(kErrInvalid, "too many windows x heads for one launch");
  const int cols = (p.N + kBlock - 1) / kBlock * kBlock;
  const int bytes = (MODE == kCols ? cols * (rows + 4) : rows * (cols + 8)) * 4;
  // the bias is kept whole as far as that leaves shared memory for the CTAs that registers allow;
  // the rows, which read it twice per window, go to three of four
  const int most = MODE == kRows || D > 16 ? 64 * 1024 : 45 * 1024;
  p.bias_pitch = bytes <= most ? cols : 0;
  const int smem = Stage<D>::FLOATS * 4 + (p.N + kTile - 1) / kTile * kTile +
                   (p.bias_pitch ? bytes
                                 : (MODE == kCols ? kTile * (rows + 4) : rows * (kTile + 8)) * 4);
  const auto kernel = grad_tf32_kernel<D, MODE>;
  static std::atomic<bool> allowed[64];  // per device
  if (int e = allow_smem(kernel, Stage<D>::MOST, allowed)) return e;
  kernel<<<unsigned(blocks), 32 * warps, smem, stream>>>(p, int(shares));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention (tf32) launch");
}

template <int D>
int launch(const Params& p, bool forward, cudaStream_t stream) {
  if (forward) return start<D, kForward>(p, stream);
  // the bias as [H, N, N], in the place of its gradient: two kernels read it, once per CTA or more
  if (int e = launch_relative_position_bias(p.dbias, kF32, p.table, kF32, p.table_rows, p.pairs,
                                            (long long)p.N * p.N, p.H, stream))
    return e;
  if (int e = start<D, kRows>(p, stream)) return e;
  if (int e = start<D, kCols>(p, stream)) return e;
  const long long warps =
      (long long)((p.N + kBlock - 1) / kBlock) * ((p.N + 15) / 16) * p.H * p.S;
  const long long blocks = (warps + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffffLL)
    return set_error(kErrInvalid, "too many windows x heads for one launch");
  if (p.vec)
    grad_bias_tf32_kernel<D, true><<<unsigned(blocks), 32 * kWarps, 0, stream>>>(p, warps);
  else
    grad_bias_tf32_kernel<D, false><<<unsigned(blocks), 32 * kWarps, 0, stream>>>(p, warps);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention gradient (tf32) launch");
}

}  // namespace

// Shares of the windows for the bias kernel: 16 warps for each of the GPU's SMs (as many as fit).
int64_t attention_grad_shares_tf32(int64_t B, int64_t H, int64_t N) {
  const int64_t tiles = (N + kBlock - 1) / kBlock * ((N + 15) / 16);
  const int64_t s = 148 * 16 / (tiles * H);
  return s < 1 ? 1 : s > B ? (B > 0 ? B : 1) : s;
}

int launch_attention_tf32(const Params& p, int head_dim, bool forward, cudaStream_t stream) {
  return head_dim == 16 ? launch<16>(p, forward, stream) : launch<32>(p, forward, stream);
}

}  // namespace crumpet
