// crumpet_b200: gradient of the window attention (fp16 / bf16, head_dim 16 or 32, N <= 352).
//
// Per window b and head h, with x = q k^T * scale + bias[h] + mask and p = softmax(x):
//   dv = p^T do,   dp = do v^T,   delta_i = sum_j p_ij dp_ij,   ds = p (dp - delta),
//   dq = ds k * scale,   dk = ds^T q * scale,   dbias[h] = sum over the windows of ds[b,h].
// Nothing of the forward pass is kept but qkv: the row statistics are taken again here, in
// fp32 and from the unrounded scores, so dbias (a sum over all windows, returned in fp32 for
// an fp32 table) is exact to fp32 rounding whatever the element type.
//
// What bounds it: one exponential per score and pass on the SFU (16 per SM and cycle) and
// about six fp32 operations per score; the products have depth head_dim = 16 or 32, a few
// percent of the tensor rate.  So the score tiles live in registers in the mma.sync fragment
// layout, where the same registers are the accumulators of one product and the operand of
// the next, rather than in tensor memory, from which every element would be read and written
// back for the arithmetic.
//
// Two kernels, each with CTAs of 64 rows x all columns of one head, which walk the windows of
// their share one after another (so what belongs to the head -- the bias, and the sum dbias
// -- stays on the SM):
//   * rows kernel (64 query rows, all keys): row statistics, dq and dbias.  Every warp holds
//     a 16 x WC tile of scores and of dp in registers (WC <= 88 keys), so each exponential is
//     taken once and the statistics (row maximum, row sum, delta) are exchanged between the
//     CG warps of a row through shared memory.  The bias tile and the dbias sums of the CTA
//     (2 x 64 x 352 fp32 = 176 KB) sit in tensor memory, used here as a second register file:
//     the bias is loaded straight into the accumulators of q k^T, dbias is read, added to and
//     written back once per window.
//   * columns kernel (64 key rows, all queries): dk and dv from the transposed scores with the
//     statistics of the first kernel; its bias tile stays in registers.
// The windows' K, V (or Q, dO) rows come in through cp.async, one window ahead.  No wait
// depends on another CTA; sums have a fixed order, so results do not change from run to run.
#include <cmath>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace crumpet {

namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRG = 4;         // row groups of 16 rows per CTA
constexpr int kBR = 16 * kRG;  // rows per CTA

struct GradParams {
  const uint16_t* qkv;   // [B, N, 3, H, HD]
  const uint16_t* dout;  // [B, N, H, HD]
  uint16_t* dqkv;        // [B, N, 3, H, HD]
  float* dbias;          // [S, H, N, N]
  float2* stats;         // [B, H, N]: (log2 of the row's sum of exponentials, delta)
  float* amax;           // [B, H, N]: largest |do| of the row (fp16 only)
  const void* table;     // [T, H]: fp32 (table_f32) or the element type
  const int* pairs;      // [N, N]: bucket of every (query, key) pair, in [0, T)
  int table_f32;
  int nwd, nwh, nww, wsd, wsh, wsw, ssd, ssh, ssw;
  int analytic;
  int B, H, N, RB, S;    // RB = row blocks, S = shares the windows are split into
  float scale;
};

// One padded token count: CG warps share a row's columns, WC columns (NT tiles of 8) each.
template <int NPAD_, int HD_>
struct Shape {
  static constexpr int NPAD = NPAD_;
  static constexpr int HD = HD_;
  static constexpr int CG = NPAD == 64 ? 1 : NPAD == 128 ? 2 : 4;
  static constexpr int WC = NPAD / CG;
  static constexpr int NT = WC / 8;
  static_assert(WC % 8 == 0 && WC <= 88, "columns per warp");
  static constexpr int WARPS = kRG * CG;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int MINB = 512 / THREADS;  // 128 registers per thread
  static constexpr int KS = HD / 16;          // depth steps of a product over the channels
  // Row pitch in shared memory: 16 bytes past the row, so the eight 16-byte rows that an
  // ldmatrix phase reads fall into different banks (pitch 48: 0, 48, 96, 16, 64, ...).
  static constexpr int PITCH = HD * 2 + 16;
  static constexpr int COLS_BYTES = NPAD * PITCH;  // one column-side tensor of a window
  static constexpr int ROWS_BYTES = kBR * PITCH;   // one row-side tensor of a window
  static constexpr int STAGE = 2 * COLS_BYTES + 2 * ROWS_BYTES;
  // tensor memory: WC/2 fp32 of bias and of dbias per thread and warp, four warps per lane
  // quarter side by side
  static constexpr int TM_WARP = WC;
  static constexpr int TM_USED = TM_WARP * CG;
  static constexpr uint32_t TM_COLS = TM_USED <= 64 ? 64 : TM_USED <= 128 ? 128
                                      : TM_USED <= 256 ? 256 : 512;
  static constexpr int RED_ROWS = WARPS * 16 * HD * 4;      // partial dq of every warp
  static constexpr int RED_COLS = 2 * WARPS * 16 * HD * 4;  // partial dk and dv
  static constexpr int EXCH = 3 * kBR * CG * 4;             // row maximum, sum, delta partials
  static constexpr int SMEM_ROWS = 2 * STAGE + RED_ROWS + EXCH + NPAD + 16;
  static constexpr int SMEM_COLS = 2 * STAGE + 2 * NPAD * 12 + RED_COLS + NPAD + 16;
  static_assert(SMEM_ROWS <= 232448 && SMEM_COLS <= 232448, "shared memory budget");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

template <bool BF16>
__device__ __forceinline__ float elem_f32(uint16_t v) {
  if constexpr (BF16) return __uint_as_float(uint32_t(v) << 16);
  else return __half2float(__ushort_as_half(v));
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// d[16x8] = a[16x16] b[16x8] + c
template <bool BF16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1, const float (&c)[4]) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
          "f"(c[2]), "f"(c[3]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
          "f"(c[2]), "f"(c[3]));
}
// d[16x8] += a[16x8] b[8x8]
template <bool BF16>
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
  else
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}

__device__ __forceinline__ void tm_ld4(uint32_t t, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3])
               : "r"(t));
}
__device__ __forceinline__ void tm_st4(uint32_t t, const float* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(t), "f"(r[0]),
               "f"(r[1]), "f"(r[2]), "f"(r[3])
               : "memory");
}
// Waits for the loads that filled `v`; the values pass through the statement, so no use of
// them can be scheduled before it.
template <int NT>
__device__ __forceinline__ void tm_wait(float (&v)[NT][4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+f"(v[t][e]));
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_wait_all() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Roll-side code of token t and the axes on which window b is the last of a shifted grid: two
// tokens of such a window belong to different regions when their codes differ there.
__device__ __forceinline__ uint32_t side_code(const GradParams& p, int t) {
  const int lw = t % p.wsw, t2 = t / p.wsw;
  const int lh = t2 % p.wsh, ld = t2 / p.wsh;
  return uint32_t(ld >= p.wsd - p.ssd) | (uint32_t(lh >= p.wsh - p.ssh) << 1) |
         (uint32_t(lw >= p.wsw - p.ssw) << 2);
}
__device__ __forceinline__ uint32_t last_axes(const GradParams& p, int b) {
  const int wi = b % (p.nwd * p.nwh * p.nww);
  const int iw = wi % p.nww, t = wi / p.nww;
  const int ih = t % p.nwh, id = t / p.nwh;
  return uint32_t(p.ssd != 0 && id == p.nwd - 1) | (uint32_t(p.ssh != 0 && ih == p.nwh - 1) << 1) |
         (uint32_t(p.ssw != 0 && iw == p.nww - 1) << 2);
}

// bias[h, i, j] / scale, as the accumulators of q k^T start; -inf past the last key, so the
// padded columns' exponentials are 0.
template <bool BF16>
__device__ __forceinline__ float bias_start(const GradParams& p, int h, int i, int j, float inv) {
  if (j >= p.N || i >= p.N) return 0.f;
  const long long t = p.pairs[(long long)i * p.N + j];
  const float v = p.table_f32
                      ? __ldg(static_cast<const float*>(p.table) + t * p.H + h)
                      : elem_f32<BF16>(__ldg(static_cast<const uint16_t*>(p.table) + t * p.H + h));
  return v * inv;
}

// Copies of `rows` token rows of one head (row stride in elements) into pitched shared memory.
template <int HD, int PITCH>
__device__ __forceinline__ void copy_rows(uint32_t dst, const uint16_t* src, long long stride,
                                          int rows, int tid, int threads) {
  constexpr int CH = HD / 8;  // 16-byte chunks per row
  for (int c = tid; c < rows * CH; c += threads) {
    const int r = c / CH, k = c % CH;
    cp16(dst + uint32_t(r * PITCH + k * 16), src + r * stride + k * 8);
  }
}

// 2^-(e + 4) for the exponent e of m: rows of do scaled by it have magnitudes below 1/8, so
// ds = p (dp - delta) of fp16 inputs stays among fp16's normal numbers whatever the loss
// scale.  1 where m is 0, subnormal or not finite.
__device__ __forceinline__ float grad_scale(float m) {
  const uint32_t e = (__float_as_uint(m) >> 23) & 0xffu;
  if (e < 24 || e > 240) return 1.f;
  return __uint_as_float((250u - e) << 23);  // 2^(127 - e - 4)
}

// ------------------------------------------------------------------------ rows kernel
template <class S, bool BF16>
__global__ void __launch_bounds__(S::THREADS, S::MINB) grad_rows_kernel(const GradParams p) {
  constexpr int NT = S::NT, HD = S::HD, CG = S::CG, PITCH = S::PITCH;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* red_b = smem + 2 * S::STAGE;
  float* red = reinterpret_cast<float*>(red_b);                      // [warp][16][HD]
  float* ex_max = reinterpret_cast<float*>(red_b + S::RED_ROWS);     // [64 rows][CG]
  float* ex_sum = ex_max + kBR * CG;
  float* ex_dp = ex_sum + kBR * CG;
  uint8_t* code = reinterpret_cast<uint8_t*>(ex_dp + kBR * CG);      // [NPAD]
  uint32_t* tm_slot = reinterpret_cast<uint32_t*>(code + S::NPAD);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rg = warp / CG, cg = warp % CG;
  const int g = lane >> 2, t4 = lane & 3;
  int blk = blockIdx.x;
  const int share = blk % p.S;
  blk /= p.S;
  const int rb = blk % p.RB, h = blk / p.RB;
  const int row0 = rb * kBR;
  const int rows = min(kBR, p.N - row0);
  const bool live = rg * 16 < rows;
  const int i0 = row0 + rg * 16 + g, i1 = i0 + 8;  // this thread's two query rows
  const int jb = cg * S::WC + 2 * t4;              // its first column; tile t adds 8 t
  const float inv_scale = 1.f / p.scale;
  const float c1 = p.scale * kLog2e;
  const float pen = -100.f * inv_scale;

  // shared memory past the window's rows stays zero
  for (int i = tid * 16; i < 2 * S::STAGE; i += S::THREADS * 16)
    *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
  if (p.analytic)
    for (int i = tid; i < S::NPAD; i += S::THREADS)
      code[i] = i < p.N ? uint8_t(side_code(p, i)) : uint8_t(0);
  if (warp == 0) {
    tmem_alloc(tm_slot, S::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // a warp reads and writes the 32 tensor-memory lanes of its quarter
  const uint32_t tm = *tm_slot + (uint32_t(32 * (warp & 3)) << 16) + uint32_t((warp >> 2) * S::TM_WARP);
  const uint32_t tm_bias = tm, tm_sum = tm + NT * 4;
  if (live) {
#pragma unroll 1
    for (int t = 0; t < NT; ++t) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = e < 2 ? i0 : i1, j = jb + 8 * t + (e & 1);
        v[e] = j < p.N ? bias_start<BF16>(p, h, i, j, inv_scale) : -INFINITY;
      }
      tm_st4(tm_bias + 4 * t, v);
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      tm_st4(tm_sum + 4 * t, z);
    }
    tmem_wait_st();
  }

  const long long tok = 3LL * p.H * HD;  // elements per token of qkv
  auto fetch = [&](int b, int st) {
    const uint32_t base = smem_u32(smem) + uint32_t(st * S::STAGE);
    const uint16_t* w = p.qkv + (long long)b * p.N * tok + h * HD;
    copy_rows<HD, PITCH>(base, w + p.H * HD, tok, p.N, tid, S::THREADS);
    copy_rows<HD, PITCH>(base + S::COLS_BYTES, w + 2 * p.H * HD, tok, p.N, tid, S::THREADS);
    copy_rows<HD, PITCH>(base + 2 * S::COLS_BYTES, w + row0 * tok, tok, rows, tid, S::THREADS);
    copy_rows<HD, PITCH>(base + 2 * S::COLS_BYTES + S::ROWS_BYTES,
                         p.dout + ((long long)b * p.N + row0) * p.H * HD + h * HD, p.H * HD, rows,
                         tid, S::THREADS);
    cp_commit();
  };

  // lane parts of the ldmatrix addresses
  const uint32_t a_off = uint32_t((lane & 15) * PITCH + (lane >> 4) * 16);             // A, rows
  const uint32_t b_off = HD == 16 ? uint32_t(((lane & 7) + (lane >> 4) * 8) * PITCH +
                                             ((lane >> 3) & 1) * 16)                   // 2 tiles
                                  : uint32_t((lane & 7) * PITCH + (lane >> 3) * 16);   // 1 tile
  const uint32_t bt_off = uint32_t((lane & 15) * PITCH + (lane >> 4) * 16);            // B, trans

  int st = 0;
  if (share < p.B) fetch(share, 0);
  for (int b = share; b < p.B; b += p.S, st ^= 1) {
    cp_wait_all();
    __syncthreads();  // window b has landed; the other stage is no longer read
    if (b + p.S < p.B) fetch(b + p.S, st ^ 1);
    if (!live) continue;
    const uint32_t ks = smem_u32(smem) + uint32_t(st * S::STAGE);
    const uint32_t vs = ks + S::COLS_BYTES;
    const uint32_t qs = vs + S::COLS_BYTES + uint32_t(rg * 16 * PITCH);
    const uint32_t gs = qs + S::ROWS_BYTES;
    const uint32_t col0 = uint32_t(cg * S::WC * PITCH);

    // scores: the accumulators start at bias / scale
    float s[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) tm_ld4(tm_bias + 4 * t, s[t]);
    {
      uint32_t a[S::KS][4];
#pragma unroll
      for (int k = 0; k < S::KS; ++k) ldsm_x4(qs + a_off + 32 * k, a[k]);
      tm_wait<NT>(s);
      if constexpr (HD == 16) {
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          uint32_t bf[4];  // past the last tile: rows of the next warp or of V, not used
          ldsm_x4(ks + col0 + uint32_t(8 * t * PITCH) + b_off, bf);
          mma16<BF16>(s[t], a[0], bf[0], bf[1], s[t]);
          if (t + 1 < NT) mma16<BF16>(s[t + 1], a[0], bf[2], bf[3], s[t + 1]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          uint32_t bf[4];
          ldsm_x4(ks + col0 + uint32_t(8 * t * PITCH) + b_off, bf);
          mma16<BF16>(s[t], a[0], bf[0], bf[1], s[t]);
          mma16<BF16>(s[t], a[1], bf[2], bf[3], s[t]);
        }
      }
    }
    if (p.analytic) {
      const uint32_t last = last_axes(p, b);
      if (last != 0) {  // padded rows (i >= N) take code 0: their results are not kept
        const uint32_t r0 = i0 < p.N ? code[i0] : 0u, r1 = i1 < p.N ? code[i1] : 0u;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t k0 = code[jb + 8 * t], k1 = code[jb + 8 * t + 1];
          if ((r0 ^ k0) & last) s[t][0] += pen;
          if ((r0 ^ k1) & last) s[t][1] += pen;
          if ((r1 ^ k0) & last) s[t][2] += pen;
          if ((r1 ^ k1) & last) s[t][3] += pen;
        }
      }
    }
    // row maxima over the CG warps of the row
    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m0 = fmaxf(m0, fmaxf(s[t][0], s[t][1]));
      m1 = fmaxf(m1, fmaxf(s[t][2], s[t][3]));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(~0u, m0, o));
      m1 = fmaxf(m1, __shfl_xor_sync(~0u, m1, o));
    }
    const int lr0 = rg * 16 + g, lr1 = lr0 + 8;
    if constexpr (CG > 1) {
      if (t4 == 0) {
        ex_max[lr0 * CG + cg] = m0;
        ex_max[lr1 * CG + cg] = m1;
      }
      bar_sync(1 + rg, 32 * CG);
#pragma unroll
      for (int c = 0; c < CG; ++c) {
        m0 = fmaxf(m0, ex_max[lr0 * CG + c]);
        m1 = fmaxf(m1, ex_max[lr1 * CG + c]);
      }
    }
    const float n0 = -m0 * c1, n1 = -m1 * c1;
    float l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t][0] = ex2(fmaf(s[t][0], c1, n0));
      s[t][1] = ex2(fmaf(s[t][1], c1, n0));
      s[t][2] = ex2(fmaf(s[t][2], c1, n1));
      s[t][3] = ex2(fmaf(s[t][3], c1, n1));
      l0 += s[t][0] + s[t][1];
      l1 += s[t][2] + s[t][3];
    }
    // dp = do v^T
    float d[NT][4];
    float g0 = 1.f, g1 = 1.f, am0 = 0.f, am1 = 0.f;
    {
      uint32_t a[S::KS][4];
#pragma unroll
      for (int k = 0; k < S::KS; ++k) ldsm_x4(gs + a_off + 32 * k, a[k]);
      if constexpr (!BF16) {  // power-of-two scale of ds, from the row's largest |do|
#pragma unroll
        for (int k = 0; k < S::KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a[k][e]));
            const float m = fmaxf(fabsf(v.x), fabsf(v.y));
            if (e & 1) am1 = fmaxf(am1, m);
            else am0 = fmaxf(am0, m);
          }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          am0 = fmaxf(am0, __shfl_xor_sync(~0u, am0, o));
          am1 = fmaxf(am1, __shfl_xor_sync(~0u, am1, o));
        }
        g0 = grad_scale(am0);
        g1 = grad_scale(am1);
      }
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (HD == 16) {
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          uint32_t bf[4];
          ldsm_x4(vs + col0 + uint32_t(8 * t * PITCH) + b_off, bf);
          mma16<BF16>(d[t], a[0], bf[0], bf[1], z);
          if (t + 1 < NT) mma16<BF16>(d[t + 1], a[0], bf[2], bf[3], z);
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          uint32_t bf[4];
          ldsm_x4(vs + col0 + uint32_t(8 * t * PITCH) + b_off, bf);
          mma16<BF16>(d[t], a[0], bf[0], bf[1], z);
          mma16<BF16>(d[t], a[1], bf[2], bf[3], d[t]);
        }
      }
    }
    float e0 = 0.f, e1 = 0.f;  // sum of p dp, before the division by the row sum
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      e0 = fmaf(s[t][0], d[t][0], e0);
      e0 = fmaf(s[t][1], d[t][1], e0);
      e1 = fmaf(s[t][2], d[t][2], e1);
      e1 = fmaf(s[t][3], d[t][3], e1);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      l0 += __shfl_xor_sync(~0u, l0, o);
      l1 += __shfl_xor_sync(~0u, l1, o);
      e0 += __shfl_xor_sync(~0u, e0, o);
      e1 += __shfl_xor_sync(~0u, e1, o);
    }
    if constexpr (CG > 1) {
      if (t4 == 0) {
        ex_sum[lr0 * CG + cg] = l0;
        ex_sum[lr1 * CG + cg] = l1;
        ex_dp[lr0 * CG + cg] = e0;
        ex_dp[lr1 * CG + cg] = e1;
      }
      bar_sync(1 + rg, 32 * CG);
      l0 = l1 = e0 = e1 = 0.f;  // every warp of the row adds the same partials in the same order
#pragma unroll
      for (int c = 0; c < CG; ++c) {
        l0 += ex_sum[lr0 * CG + c];
        l1 += ex_sum[lr1 * CG + c];
        e0 += ex_dp[lr0 * CG + c];
        e1 += ex_dp[lr1 * CG + c];
      }
    }
    const float inv0 = 1.f / l0, inv1 = 1.f / l1;
    const float del0 = e0 * inv0, del1 = e1 * inv1;
    if (cg == 0 && t4 == 0) {  // statistics for the columns kernel
      const long long at = ((long long)b * p.H + h) * p.N;
      if (i0 < p.N) p.stats[at + i0] = make_float2(fmaf(m0, c1, log2f(l0)), del0);
      if (i1 < p.N) p.stats[at + i1] = make_float2(fmaf(m1, c1, log2f(l1)), del1);
      if constexpr (!BF16) {
        if (i0 < p.N) p.amax[at + i0] = am0;
        if (i1 < p.N) p.amax[at + i1] = am1;
      }
    }
    // ds = p (dp - delta), in place of dp
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      d[t][0] = (d[t][0] - del0) * (s[t][0] * inv0);
      d[t][1] = (d[t][1] - del0) * (s[t][1] * inv0);
      d[t][2] = (d[t][2] - del1) * (s[t][2] * inv1);
      d[t][3] = (d[t][3] - del1) * (s[t][3] * inv1);
    }
    // dbias += ds
    tmem_wait_st();  // the previous window's sums are written
#pragma unroll
    for (int t = 0; t < NT; ++t) tm_ld4(tm_sum + 4 * t, s[t]);
    tm_wait<NT>(s);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] += d[t][e];
      tm_st4(tm_sum + 4 * t, s[t]);
    }
    // dq = ds k, ds rounded to the element type (scaled as above): the rounding errors of a
    // row's keys are independent, so they add up like one rounding of dq itself
    float acc[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      uint32_t a[4];
      a[0] = pack2<BF16>(d[t][0] * g0, d[t][1] * g0);
      a[1] = pack2<BF16>(d[t][2] * g1, d[t][3] * g1);
      if (t + 1 < NT) {
        a[2] = pack2<BF16>(d[t + 1][0] * g0, d[t + 1][1] * g0);
        a[3] = pack2<BF16>(d[t + 1][2] * g1, d[t + 1][3] * g1);
      }
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) {
        uint32_t bf[4];  // past the last tile: as above
        ldsm_x4_t(ks + col0 + uint32_t(8 * t * PITCH) + bt_off + 32 * n, bf);
        if (t + 1 < NT) {
          mma16<BF16>(acc[2 * n], a, bf[0], bf[1], acc[2 * n]);
          mma16<BF16>(acc[2 * n + 1], a, bf[2], bf[3], acc[2 * n + 1]);
        } else {
          mma8<BF16>(acc[2 * n], a[0], a[1], bf[0]);
          mma8<BF16>(acc[2 * n + 1], a[0], a[1], bf[2]);
        }
      }
    }
    const float f0 = BF16 ? p.scale : p.scale / g0, f1 = BF16 ? p.scale : p.scale / g1;
    float* mine = red + (rg * CG + cg) * 16 * HD;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      *reinterpret_cast<float2*>(mine + g * HD + 8 * n + 2 * t4) =
          make_float2(acc[n][0] * f0, acc[n][1] * f0);
      *reinterpret_cast<float2*>(mine + (g + 8) * HD + 8 * n + 2 * t4) =
          make_float2(acc[n][2] * f1, acc[n][3] * f1);
    }
    bar_sync(1 + rg, 32 * CG);
    const float* all = red + rg * CG * 16 * HD;
    for (int o = cg * 32 + lane; o < 16 * HD / 2; o += 32 * CG) {
      const int r = o / (HD / 2), c = (o % (HD / 2)) * 2;
      float2 v = *reinterpret_cast<const float2*>(all + r * HD + c);
#pragma unroll
      for (int k = 1; k < CG; ++k) {
        const float2 w = *reinterpret_cast<const float2*>(all + k * 16 * HD + r * HD + c);
        v.x += w.x;
        v.y += w.y;
      }
      const int i = row0 + rg * 16 + r;
      if (i < p.N)
        *reinterpret_cast<uint32_t*>(p.dqkv + ((long long)b * p.N + i) * tok + h * HD + c) =
            pack2<BF16>(v.x, v.y);
    }
  }

  if (live) {  // the head's dbias of this share of the windows
    tmem_wait_st();
    float* out = p.dbias + ((long long)share * p.H + h) * p.N * p.N;
#pragma unroll 1
    for (int t = 0; t < NT; ++t) {
      float v[1][4];
      tm_ld4(tm_sum + 4 * t, v[0]);
      tm_wait<1>(v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = e < 2 ? i0 : i1, j = jb + 8 * t + (e & 1);
        if (i < p.N && j < p.N) out[(long long)i * p.N + j] = v[0][e];
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(*tm_slot, S::TM_COLS);
  }
}

// --------------------------------------------------------------------- columns kernel
// The same tiles transposed: rows are 64 keys, columns all queries; p and ds come from the
// statistics, are rounded and multiplied by do and q at once, two tiles at a time.
template <class S, bool BF16>
__global__ void __launch_bounds__(S::THREADS, S::MINB) grad_cols_kernel(const GradParams p) {
  constexpr int NT = S::NT, HD = S::HD, CG = S::CG, PITCH = S::PITCH;
  extern __shared__ __align__(16) uint8_t smem[];
  float2* stat_s = reinterpret_cast<float2*>(smem + 2 * S::STAGE);      // [2][NPAD]
  float* amax_s = reinterpret_cast<float*>(stat_s + 2 * S::NPAD);       // [2][NPAD]
  float* red = amax_s + 2 * S::NPAD;                                    // [2][warp][16][HD]
  uint8_t* code = reinterpret_cast<uint8_t*>(red) + S::RED_COLS;        // [NPAD]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rg = warp / CG, cg = warp % CG;
  const int g = lane >> 2, t4 = lane & 3;
  int blk = blockIdx.x;
  const int share = blk % p.S;
  blk /= p.S;
  const int rb = blk % p.RB, h = blk / p.RB;
  const int row0 = rb * kBR;
  const int rows = min(kBR, p.N - row0);
  const bool live = rg * 16 < rows;
  const int k0 = row0 + rg * 16 + g, k1 = k0 + 8;  // this thread's two keys
  const int ib = cg * S::WC + 2 * t4;              // its first query; tile t adds 8 t
  const float inv_scale = 1.f / p.scale;
  const float c1 = p.scale * kLog2e;
  const float pen = -100.f * inv_scale;

  // zero past the window's rows: Q, dO, K, V and the statistics
  for (int i = tid * 16; i < 2 * S::STAGE + 2 * S::NPAD * 12; i += S::THREADS * 16)
    *reinterpret_cast<uint4*>(smem + i) = make_uint4(0, 0, 0, 0);
  if (p.analytic)
    for (int i = tid; i < S::NPAD; i += S::THREADS)
      code[i] = i < p.N ? uint8_t(side_code(p, i)) : uint8_t(0);
  __syncthreads();

  float bias[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = e < 2 ? k0 : k1, i = ib + 8 * t + (e & 1);
      bias[t][e] = i < p.N ? bias_start<BF16>(p, h, i, k, inv_scale) : -INFINITY;
    }

  const long long tok = 3LL * p.H * HD;
  auto fetch = [&](int b, int st) {
    const uint32_t base = smem_u32(smem) + uint32_t(st * S::STAGE);
    const uint16_t* w = p.qkv + (long long)b * p.N * tok + h * HD;
    copy_rows<HD, PITCH>(base, w, tok, p.N, tid, S::THREADS);
    copy_rows<HD, PITCH>(base + S::COLS_BYTES, p.dout + (long long)b * p.N * p.H * HD + h * HD,
                         p.H * HD, p.N, tid, S::THREADS);
    copy_rows<HD, PITCH>(base + 2 * S::COLS_BYTES, w + p.H * HD + row0 * tok, tok, rows, tid,
                         S::THREADS);
    copy_rows<HD, PITCH>(base + 2 * S::COLS_BYTES + S::ROWS_BYTES, w + 2 * p.H * HD + row0 * tok,
                         tok, rows, tid, S::THREADS);
    const long long at = ((long long)b * p.H + h) * p.N;
    for (int i = tid; i < p.N; i += S::THREADS) {
      cp8(smem_u32(stat_s + st * S::NPAD + i), p.stats + at + i);
      if constexpr (!BF16) cp4(smem_u32(amax_s + st * S::NPAD + i), p.amax + at + i);
    }
    cp_commit();
  };

  const uint32_t a_off = uint32_t((lane & 15) * PITCH + (lane >> 4) * 16);
  const uint32_t b_off = HD == 16 ? uint32_t(((lane & 7) + (lane >> 4) * 8) * PITCH +
                                             ((lane >> 3) & 1) * 16)
                                  : uint32_t((lane & 7) * PITCH + (lane >> 3) * 16);
  const uint32_t bt_off = uint32_t((lane & 15) * PITCH + (lane >> 4) * 16);

  int st = 0;
  if (share < p.B) fetch(share, 0);
  for (int b = share; b < p.B; b += p.S, st ^= 1) {
    cp_wait_all();
    __syncthreads();
    if (b + p.S < p.B) fetch(b + p.S, st ^ 1);
    if (!live) continue;
    const uint32_t qs = smem_u32(smem) + uint32_t(st * S::STAGE);
    const uint32_t gs = qs + S::COLS_BYTES;
    const uint32_t ks = gs + S::COLS_BYTES + uint32_t(rg * 16 * PITCH);
    const uint32_t vs = ks + S::ROWS_BYTES;
    const uint32_t col0 = uint32_t(cg * S::WC * PITCH);
    const float2* stat = stat_s + st * S::NPAD;

    // one power-of-two scale of ds for the window (fp16): its sum over the queries goes
    // through one accumulator
    float gscale = 1.f;
    if constexpr (!BF16) {
      float m = 0.f;
      for (int i = lane; i < S::NPAD; i += 32) m = fmaxf(m, amax_s[st * S::NPAD + i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
      gscale = grad_scale(m);
    }
    uint32_t last = 0;
    if (p.analytic) last = last_axes(p, b);
    const uint32_t r0 = last && k0 < p.N ? code[k0] : 0u, r1 = last && k1 < p.N ? code[k1] : 0u;

    uint32_t ka[S::KS][4], va[S::KS][4];
#pragma unroll
    for (int k = 0; k < S::KS; ++k) {
      ldsm_x4(ks + a_off + 32 * k, ka[k]);
      ldsm_x4(vs + a_off + 32 * k, va[k]);
    }
    float dk[HD / 8][4], dv[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;

#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      constexpr float z[4] = {0.f, 0.f, 0.f, 0.f};
      uint32_t pa[4], da[4];
      uint32_t bq[4], bg[4];
      if constexpr (HD == 16) {
        ldsm_x4(qs + col0 + uint32_t(8 * t * PITCH) + b_off, bq);
        ldsm_x4(gs + col0 + uint32_t(8 * t * PITCH) + b_off, bg);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t + u >= NT) break;
        float s[4], d[4];
        if constexpr (HD == 16) {
          mma16<BF16>(s, ka[0], bq[2 * u], bq[2 * u + 1], bias[t + u]);
          mma16<BF16>(d, va[0], bg[2 * u], bg[2 * u + 1], z);
        } else {
          ldsm_x4(qs + col0 + uint32_t(8 * (t + u) * PITCH) + b_off, bq);
          ldsm_x4(gs + col0 + uint32_t(8 * (t + u) * PITCH) + b_off, bg);
          mma16<BF16>(s, ka[0], bq[0], bq[1], bias[t + u]);
          mma16<BF16>(s, ka[1], bq[2], bq[3], s);
          mma16<BF16>(d, va[0], bg[0], bg[1], z);
          mma16<BF16>(d, va[1], bg[2], bg[3], d);
        }
        const int i = ib + 8 * (t + u);
        if (last) {
          const uint32_t c0 = code[i], c1_ = code[i + 1];
          if ((r0 ^ c0) & last) s[0] += pen;
          if ((r0 ^ c1_) & last) s[1] += pen;
          if ((r1 ^ c0) & last) s[2] += pen;
          if ((r1 ^ c1_) & last) s[3] += pen;
        }
        const float4 x = *reinterpret_cast<const float4*>(stat + i);  // two queries' statistics
        float q[4];
        q[0] = ex2(fmaf(s[0], c1, -x.x));
        q[1] = ex2(fmaf(s[1], c1, -x.z));
        q[2] = ex2(fmaf(s[2], c1, -x.x));
        q[3] = ex2(fmaf(s[3], c1, -x.z));
        d[0] = (d[0] - x.y) * q[0];
        d[1] = (d[1] - x.w) * q[1];
        d[2] = (d[2] - x.y) * q[2];
        d[3] = (d[3] - x.w) * q[3];
        if constexpr (!BF16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] *= gscale;
        }
        pa[2 * u] = pack2<BF16>(q[0], q[1]);
        pa[2 * u + 1] = pack2<BF16>(q[2], q[3]);
        da[2 * u] = pack2<BF16>(d[0], d[1]);
        da[2 * u + 1] = pack2<BF16>(d[2], d[3]);
      }
#pragma unroll
      for (int n = 0; n < HD / 16; ++n) {
        uint32_t tq[4], tg[4];
        ldsm_x4_t(gs + col0 + uint32_t(8 * t * PITCH) + bt_off + 32 * n, tg);
        ldsm_x4_t(qs + col0 + uint32_t(8 * t * PITCH) + bt_off + 32 * n, tq);
        if (t + 1 < NT) {
          mma16<BF16>(dv[2 * n], pa, tg[0], tg[1], dv[2 * n]);
          mma16<BF16>(dv[2 * n + 1], pa, tg[2], tg[3], dv[2 * n + 1]);
          mma16<BF16>(dk[2 * n], da, tq[0], tq[1], dk[2 * n]);
          mma16<BF16>(dk[2 * n + 1], da, tq[2], tq[3], dk[2 * n + 1]);
        } else {
          mma8<BF16>(dv[2 * n], pa[0], pa[1], tg[0]);
          mma8<BF16>(dv[2 * n + 1], pa[0], pa[1], tg[2]);
          mma8<BF16>(dk[2 * n], da[0], da[1], tq[0]);
          mma8<BF16>(dk[2 * n + 1], da[0], da[1], tq[2]);
        }
      }
    }
    const float f = BF16 ? p.scale : p.scale / gscale;
    float* mk = red + (rg * CG + cg) * 16 * HD;
    float* mv = mk + S::WARPS * 16 * HD;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      const int o0 = g * HD + 8 * n + 2 * t4, o1 = (g + 8) * HD + 8 * n + 2 * t4;
      *reinterpret_cast<float2*>(mk + o0) = make_float2(dk[n][0] * f, dk[n][1] * f);
      *reinterpret_cast<float2*>(mk + o1) = make_float2(dk[n][2] * f, dk[n][3] * f);
      *reinterpret_cast<float2*>(mv + o0) = make_float2(dv[n][0], dv[n][1]);
      *reinterpret_cast<float2*>(mv + o1) = make_float2(dv[n][2], dv[n][3]);
    }
    bar_sync(1 + rg, 32 * CG);
    for (int o = cg * 32 + lane; o < 16 * HD; o += 32 * CG) {
      const int w = o / (8 * HD), r = (o / (HD / 2)) % 16, c = (o % (HD / 2)) * 2;
      const float* all = red + w * S::WARPS * 16 * HD + rg * CG * 16 * HD + r * HD + c;
      float2 v = *reinterpret_cast<const float2*>(all);
#pragma unroll
      for (int k = 1; k < CG; ++k) {
        const float2 a = *reinterpret_cast<const float2*>(all + k * 16 * HD);
        v.x += a.x;
        v.y += a.y;
      }
      const int i = row0 + rg * 16 + r;
      if (i < p.N)
        *reinterpret_cast<uint32_t*>(p.dqkv + ((long long)b * p.N + i) * tok +
                                     (long long)(1 + w) * p.H * HD + h * HD + c) =
            pack2<BF16>(v.x, v.y);
    }
  }
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

template <class S, bool BF16>
int launch_grad(const GradParams& p, cudaStream_t stream) {
  static bool configured[64] = {false};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(grad_rows_kernel<S, BF16>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         S::SMEM_ROWS);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(grad_cols_kernel<S, BF16>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_COLS);
    if (e != cudaSuccess) return set_cuda_error(e, "attention gradient smem attribute");
    if (dev < 64) configured[dev] = true;
  }
  const unsigned blocks = unsigned(p.H) * unsigned(p.RB) * unsigned(p.S);
  grad_rows_kernel<S, BF16><<<blocks, S::THREADS, S::SMEM_ROWS, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "attention gradient (rows) launch");
  grad_cols_kernel<S, BF16><<<blocks, S::THREADS, S::SMEM_COLS, stream>>>(p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "attention gradient (columns) launch");
  return kOk;
}

template <int HD, bool BF16>
int dispatch_npad(const GradParams& p, cudaStream_t stream) {
  if (p.N <= 64) return launch_grad<Shape<64, HD>, BF16>(p, stream);
  if (p.N <= 128) return launch_grad<Shape<128, HD>, BF16>(p, stream);
  if (p.N <= 224) return launch_grad<Shape<224, HD>, BF16>(p, stream);
  return launch_grad<Shape<352, HD>, BF16>(p, stream);
}

}  // namespace

bool attention_grad_tensor_path(int dtype, int64_t N, int64_t head_dim) {
  return dtype != kF32 && (head_dim == 16 || head_dim == 32) && N >= 1 && N <= 352;
}

// Shares the windows are split into: as many as keep every SM's CTA slots busy with one CTA
// per (head, row block, share), at most one per window.
int64_t attention_grad_shares(int64_t B, int64_t H, int64_t N) {
  const int64_t per_sm = N <= 64 ? 4 : N <= 128 ? 2 : 1;
  const int64_t blocks = H * ((N + kBR - 1) / kBR);
  const int64_t s = int64_t(sm_count()) * per_sm / blocks;
  return s < 1 ? 1 : s > B ? (B > 0 ? B : 1) : s;
}

int launch_attention_grad(const AttnGradArgs& a, cudaStream_t stream) {
  GradParams p{};
  p.qkv = static_cast<const uint16_t*>(a.qkv);
  p.dout = static_cast<const uint16_t*>(a.grad_out);
  p.dqkv = static_cast<uint16_t*>(a.grad_qkv);
  p.dbias = a.grad_bias;
  p.stats = reinterpret_cast<float2*>(a.stats);
  p.amax = a.stats + 2 * a.B * a.H * a.N;
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
  p.RB = int((a.N + kBR - 1) / kBR);
  p.S = int(a.shares);
  p.scale = a.scale;
  const bool bf16 = a.dtype == kBF16;
  if (a.head_dim == 32)
    return bf16 ? dispatch_npad<32, true>(p, stream) : dispatch_npad<32, false>(p, stream);
  return bf16 ? dispatch_npad<16, true>(p, stream) : dispatch_npad<16, false>(p, stream);
}

}  // namespace crumpet
