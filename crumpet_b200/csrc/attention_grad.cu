// crumpet_b200: gradient of the window attention (fp16 / bf16, head_dim 16 or 32, N <= 352).
//
// Per window b and head h, with x = q k^T * scale + bias[h] + mask and p = softmax(x):
//   dv = p^T do,   dp = do v^T,   delta_i = sum_j p_ij dp_ij,   ds = p (dp - delta),
//   dq = ds k * scale,   dk = ds^T q * scale,   dbias[h] = sum over the windows of ds[b,h].
// Nothing of the forward pass is kept but qkv: the row statistics are taken again here, in
// fp32 and from unrounded scores, so dbias (a sum over all windows, returned in fp32 for an fp32
// table) is the gradient at the table's own values to fp32 rounding, whatever the element type.
// (The forward rounds an fp32 table's bias to the element type for its tensor-core operand,
// scores moved by up to 2^-8 |bias| in bf16; kept unrounded there it would take a second operand
// as large as the first.)
//
// What bounds it: one exponential per score and pass on the SFU (16 per SM and cycle) and
// about six fp32 operations per score; the products have depth head_dim = 16 or 32, a few
// percent of the tensor rate.  So the score tiles live in registers in the mma.sync fragment
// layout, where the same registers are the accumulators of one product and the operand of
// the next, rather than in tensor memory, from which every element would be read and written
// back for the arithmetic.
//
// Two kernels; a CTA takes some rows x all columns of one head and walks the windows of its
// share one after another, so what belongs to the head -- the bias, and the sum dbias -- stays
// on the SM, in tensor memory, used here as a second register file:
//   * rows kernel (64 query rows, all keys): row statistics, dq and dbias.  A warp holds a
//     16 x WC tile of scores in registers (WC <= 88 keys), so each exponential is taken once (dp,
//     one product, twice); the CG warps of a row exchange (maximum, sum, sum of p dp) through shared
//     memory at one barrier per window, behind which they also join the dq of the window
//     before.  The bias goes from tensor memory straight into the accumulators of q k^T; dbias
//     is read from it, added to and written back once per window (2 x 64 x 352 fp32).
//   * columns kernel: dk and dv from the transposed scores with the statistics of the first
//     kernel; a warp takes 16 keys x all queries, so nothing is exchanged between warps.
// TMA brings the windows' rows into a ring of stages; the last warp that has read a stage
// refills it, so warps drift apart by up to a ring and no warp waits only to copy.  Waits for
// the loads are bounded like the forward kernel's (2 s, then the device error word).  No wait
// depends on another CTA; sums have a fixed order, so results do not change from run to run.
//
// Measured, three heads of 16 channels and 343 tokens: 1372 windows in bf16 rows 557 us, columns
// 321 us (the exponentials alone 117 us each, with the padding); 343 windows in fp16 162 and 107
// us, issue slots 42 % and 34 % busy: latency bounds both, in the rows kernel that of the exchange
// between the warps of a row (its largest stall; one row group alone on an SM takes 348 of 571
// us).  Nearly all columns kernels and the rows kernels of the widest shapes spill (8 to 100 bytes
// per thread, at 128 to 168 registers).  Measured and not kept in the rows kernel, against 571 us:
// dp held in registers as well (595 to 661 us), two windows' halves in flight (740 us, registers
// spill).
#include <cmath>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace crumpet {

static __device__ int g_grad_error;  // 1: a bounded wait expired, 2: a bucket out of range

namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRG = 4;         // row groups of 16 rows per CTA of the rows kernel
constexpr int kBR = 16 * kRG;  // its rows
constexpr int kSmemBudget = 227 * 1024 - 1024;  // per SM, less what the CTAs reserve

struct GradParams {
  uint16_t* dqkv;        // [B, N, 3, H, HD]
  float* dbias;          // [S, H, N, N]
  float* stats;          // [B, H, NS / 2][4]: of two rows, -log2 of the sums of exponentials, -deltas
  float* amax;           // [B, H, groups of 16 rows]: their largest |do| (fp16 only)
  const void* table;     // [T, H]: fp32 (table_f32) or the element type
  const int* pairs;      // [N, N]: bucket of every (query, key) pair
  int table_f32, table_rows;  // a bucket outside [0, table_rows) is flagged and adds no bias
  int nwd, nwh, nww, wsd, wsh, wsw, ssd, ssh, ssw;
  int analytic;
  uint32_t mask_pen, mask_one;  // the mask features' values (MaskPenalty)
  int B, H, N, NS;       // NS = N rounded up to 2: rows of stats start on 16 bytes
  int RB, S;             // row blocks, and shares that the windows are split into
  float scale;
};

// What both kernels share: token rows in shared memory as TMA writes them, HD * 2 bytes each in
// the 32- or 64-byte swizzle, whose permuted 16-byte chunks let eight rows of an ldmatrix phase
// fall into different banks.
template <int HD>
struct Rows {
  static constexpr int BYTES = HD * 2;
  static constexpr int KS = HD / 16;  // depth steps of a product over the channels
  // offset of 16-byte chunk c of row r, for rows counted from a multiple of 8
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    const int sw = HD == 16 ? (r >> 2) & 1 : (r >> 1) & 3;
    return uint32_t(r * BYTES + ((c ^ sw) << 4));
  }
};

// Boxes of a TMA load of `rows` token rows: equal, at most 256 rows.
__host__ __device__ constexpr int box_rows(int rows) { return rows > 256 ? rows / 2 : rows; }

// Rows kernel: CG warps share a row's NPAD columns, WC columns (NT tiles of 8) each.
template <int NPAD_, int HD_>
struct RowsShape {
  static constexpr int NPAD = NPAD_, HD = HD_;
  static constexpr int CG = NPAD == 64 ? 1 : NPAD == 128 ? 2 : 4;
  static constexpr int WC = NPAD / CG;
  static constexpr int NT = WC / 8;
  static_assert(WC % 8 == 0 && WC <= 88, "columns per warp");
  static constexpr int WARPS = kRG * CG;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int MINB = 512 / THREADS;  // 128 registers per thread
  static constexpr int COLS = NPAD * HD * 2;  // bytes of K or V of a window
  static constexpr int ROWS = kBR * HD * 2;   // bytes of the CTA's rows of Q or dO
  static constexpr int STAGE = 2 * COLS + 2 * ROWS;
  // tensor memory: WC/2 fp32 of bias and of dbias per thread and warp, the CG warps of a lane
  // quarter side by side
  static constexpr int TM_USED = WC * CG;
  static constexpr uint32_t TM_COLS = TM_USED <= 64 ? 64 : TM_USED <= 128 ? 128
                                      : TM_USED <= 256 ? 256 : 512;
  static constexpr int PITCH = HD + 8;                      // floats per row of partial dq
  static constexpr int RED = 2 * WARPS * 16 * PITCH * 4;    // partial dq, two windows
  static constexpr int EXCH = 2 * CG * kBR * 16;            // row statistics, two windows
  static constexpr int MASK = NPAD * 16;                    // mask features of the columns
  static constexpr int FIXED = RED + EXCH + MASK + 1024 + 256;
  static constexpr int FIT = (kSmemBudget / MINB - FIXED) / STAGE;
  static constexpr int STAGES = FIT > 4 ? 4 : FIT;
  static constexpr int SMEM = STAGES * STAGE + FIXED;
  static_assert(STAGES >= 2 && SMEM <= 232448, "shared memory budget");
};

// Columns kernel: a warp takes 16 keys and all NPAD queries, NT tiles of 8.
template <int NPAD_, int HD_>
struct ColsShape {
  static constexpr int NPAD = NPAD_, HD = HD_;
  static constexpr int NT = NPAD / 8;
  static_assert(NT % 2 == 0, "tiles are taken in pairs");
  static constexpr int WARPS = NPAD == 352 ? 11 : NPAD == 224 ? 7 : 4;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int MINB = NPAD == 352 ? 1 : NPAD == 224 ? 2 : 4;  // CTAs per SM
  static constexpr int BR = 16 * WARPS;  // rows (keys) per CTA
  // Tensor memory: 4 fp32 of the bias per thread and tile, the warps of a lane quarter side by
  // side; the tiles that do not fit stay in registers (2 of 44 where three warps share 512).
  static constexpr int QUARTER = (WARPS + 3) / 4;
  static constexpr int TT = 512 / MINB / (4 * QUARTER) < NT ? 512 / MINB / (4 * QUARTER) / 2 * 2 : NT;
  static constexpr int TM_USED = 4 * TT * QUARTER;
  static constexpr uint32_t TM_COLS = TM_USED <= 32 ? 32 : TM_USED <= 64 ? 64
                                      : TM_USED <= 128 ? 128 : TM_USED <= 256 ? 256 : 512;
  static_assert(TM_COLS * MINB <= 512 && NT - TT <= 2, "tensor memory budget");
  static constexpr int COLS = NPAD * HD * 2;  // bytes of Q or dO of a window
  static constexpr int ROWS = BR * HD * 2;    // bytes of the CTA's rows of K or V
  static constexpr int STAT = NPAD * 8;       // statistics of the window's rows
  static constexpr int STAGE = (2 * COLS + 2 * ROWS + STAT + 1023) / 1024 * 1024;
  static constexpr int MASK = NPAD * 16;
  static constexpr int FIXED = MASK + 1024 + 256;
  static constexpr int FIT = (kSmemBudget / MINB - FIXED) / STAGE;
  static constexpr int STAGES = FIT > 4 ? 4 : FIT;
  static constexpr int SMEM = STAGES * STAGE + FIXED;
  static_assert(STAGES >= 2 && SMEM <= 232448, "shared memory budget");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {  // within 1 ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// 4 NT consecutive tensor-memory columns of this thread's lane (widths are powers of two)
template <int N>
__device__ __forceinline__ void tm_ld(uint32_t t, float* r) {
  if constexpr (N >= 32) {
    tmem_ld32(t, reinterpret_cast<uint32_t*>(r));
    tm_ld<N - 32>(t + 32, r + 32);
  } else if constexpr (N >= 16) {
    tmem_ld16(t, reinterpret_cast<uint32_t(&)[16]>(*r));
    tm_ld<N - 16>(t + 16, r + 16);
  } else if constexpr (N >= 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]),
                   "=f"(r[6]), "=f"(r[7])
                 : "r"(t));
    tm_ld<N - 8>(t + 8, r + 8);
  } else if constexpr (N >= 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3])
                 : "r"(t));
    tm_ld<N - 4>(t + 4, r + 4);
  }
}
template <int N>
__device__ __forceinline__ void tm_st(uint32_t t, const float* r) {
  if constexpr (N >= 32) {
    tmem_st32(t, reinterpret_cast<const uint32_t*>(r));
    tm_st<N - 32>(t + 32, r + 32);
  } else if constexpr (N >= 16) {
    tmem_st16(t, reinterpret_cast<const uint32_t*>(r));
    tm_st<N - 16>(t + 16, r + 16);
  } else if constexpr (N >= 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t),
                 "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]),
                 "f"(r[7])
                 : "memory");
    tm_st<N - 8>(t + 8, r + 8);
  } else if constexpr (N >= 4) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(t), "f"(r[0]),
                 "f"(r[1]), "f"(r[2]), "f"(r[3])
                 : "memory");
    tm_st<N - 4>(t + 4, r + 4);
  }
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// The two values of a row in a fragment, for the packed fp32 arithmetic (two per instruction)
__device__ __forceinline__ float2 two(const float (&v)[4], int row) {
  return make_float2(v[2 * row], v[2 * row + 1]);
}
__device__ __forceinline__ void put(float (&v)[4], int row, float2 x) {
  v[2 * row] = x.x;
  v[2 * row + 1] = x.y;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Untiled copy global -> shared (16-byte aligned, a multiple of 16 bytes), counted on `bar`
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
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

// The accumulators that q k^T starts from: bias[h, i, j] / scale, -inf past the last column (its
// exponentials are 0), 0 in padded rows.  `at(t, e)` gives the (query, key) of a value; two rounds
// of independent gathers, since a CTA does nothing else meanwhile.
template <int NT, bool BF16, bool COLS>
__device__ __forceinline__ void start_values(const GradParams& p, int h, int row0, int col0,
                                             float (&v)[NT][4]) {
  int at[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = row0 + (e < 2 ? 0 : 8), c = col0 + 8 * t + (e & 1);
      at[t][e] = r < p.N && c < p.N ? __ldg(p.pairs + (COLS ? c * p.N + r : r * p.N + c)) : 0;
    }
  bool bad = false;
  const float inv = 1.f / p.scale;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = row0 + (e < 2 ? 0 : 8), c = col0 + 8 * t + (e & 1);
      float x = c < p.N ? 0.f : -INFINITY;
      const bool inside = unsigned(at[t][e]) < unsigned(p.table_rows);
      bad = bad || !inside;
      if (inside && r < p.N && c < p.N) {
        const long long i = (long long)at[t][e] * p.H + h;
        x = inv * (p.table_f32 ? __ldg(static_cast<const float*>(p.table) + i)
                               : elem_f32<BF16>(__ldg(static_cast<const uint16_t*>(p.table) + i)));
      }
      v[t][e] = x;
    }
  if (bad) atomicOr(&g_grad_error, 2);
}

// Shifted-window mask as one more product of depth 8 in the windows that need it, over the eight
// roll-side codes: a column token has the feature mask_one at its own code, a row token mask_pen at
// the codes that differ from its own on one of the window's masked axes `last`, so a pair gets their
// product -100 / scale once, on however many axes it differs.  Element pairs (codes 2 t4 and
// 2 t4 + 1) as mma operands.
__device__ __forceinline__ uint32_t row_feature(uint32_t pen, uint32_t code, uint32_t last, int t4) {
  const uint32_t apart = (uint32_t(2 * t4) ^ code) & last;  // of code 2 t4; the other's bit 0 differs
  return (apart ? pen : 0u) | ((apart ^ (last & 1u)) ? pen << 16 : 0u);
}
__device__ __forceinline__ uint32_t col_feature(uint32_t one, uint32_t code, int t4) {
  return int(code >> 1) != t4 ? 0u : (code & 1u) ? one << 16 : one;
}

// 2^-(e + 4) for the exponent e of m: rows of do scaled by it have magnitudes below 1/8, so
// ds = p (dp - delta) of fp16 inputs stays among fp16's normal numbers whatever the loss
// scale.  1 where m is 0, subnormal or not finite.
__device__ __forceinline__ float grad_scale(float m) {
  const uint32_t e = (__float_as_uint(m) >> 23) & 0xffu;
  if (e < 24 || e > 240) return 1.f;
  return __uint_as_float((250u - e) << 23);  // 2^(127 - e - 4)
}

__device__ __forceinline__ float inverse_scale(float g) {  // 1 / g of a power of two
  return __uint_as_float((254u << 23) - __float_as_uint(g));
}

// ------------------------------------------------------------------- ring of windows
// The CTA's windows k = 0, 1, ... (window share + k S of the batch) pass through STAGES stages of
// shared memory.  One thread issues a window's loads; the warps wait for its stage to be full,
// and the last warp to have read a stage issues the window that comes next in it.
constexpr int kMaxStages = 4;
struct Tail {  // the CTA's shared words
  uint64_t full[kMaxStages];
  uint32_t done[kMaxStages];  // warps that have read the stage
  uint32_t last[kMaxStages];  // the stage's window: axes with a roll seam (last_axes)
  uint32_t tm_slot;
  int abort;   // a wait expired: no more waiting, no more loads
  int issued;  // windows whose loads were issued
};

__device__ __forceinline__ void init_tail(Tail* tail) {
  for (int s = 0; s < kMaxStages; ++s) {
    mbar_init(&tail->full[s], 1);
    tail->done[s] = 0;
  }
  tail->abort = 0;
  tail->issued = 0;
  fence_mbar_init();
}

// Whether the stage of window k is full.  After a wait has expired the warps go on without
// waiting, so they keep meeting at their barriers; what they compute is not used.
template <int STAGES>
__device__ __forceinline__ void wait_stage(Tail* tail, int k) {
  mbar_wait(&tail->full[k % STAGES], uint32_t(k / STAGES) & 1u, &tail->abort);
  __syncwarp();
}

// Counts this warp's reading of window k as finished; true for the lane that now has to issue
// window k + STAGES.
template <int STAGES>
__device__ __forceinline__ bool release_stage(Tail* tail, int k, int count, uint32_t warps) {
  __syncwarp();
  if ((threadIdx.x & 31) != 0) return false;
  __threadfence_block();  // this warp's reads come before the loads that follow the count
  if (atomicAdd(&tail->done[k % STAGES], 1u) + 1u != warps) return false;
  tail->done[k % STAGES] = 0;
  __threadfence_block();
  return k + STAGES < count && *reinterpret_cast<volatile int*>(&tail->abort) == 0;
}

// After the CTA's last barrier, by one thread: reports an expired wait, and lets loads that are
// still in flight land (bounded) before the CTA's shared memory is given back.
template <int STAGES>
__device__ __forceinline__ void finish_ring(Tail* tail) {
  if (tail->abort == 0) return;
  atomicOr(&g_grad_error, 1);
  for (int k = tail->issued - 1; k >= 0 && k >= tail->issued - STAGES; --k) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(&tail->full[k % STAGES], uint32_t(k / STAGES) & 1u))
      if (globaltimer_ns() - t0 > kWaitLimitNs) break;
  }
}

// TMA loads of ROWS token rows from row0 of (head h, window b), in equal boxes
template <int HD, int ROWS>
__device__ __forceinline__ void load_rows(uint8_t* dst, const CUtensorMap* map, uint64_t* full,
                                          int row0, int h, int b) {
#pragma unroll
  for (int r = 0; r < ROWS; r += box_rows(ROWS))
    tma_load_4d(dst + r * HD * 2, map, full, 0, row0 + r, h, b);
}

// The tensors that a kernel loads: two in boxes of all the window's tokens, two of the CTA's rows
// (rows kernel: k, v and q, do; columns kernel: q, do and k, v).
struct Maps {
  CUtensorMap cols0, cols1, rows0, rows1;
};

// ------------------------------------------------------------------------ rows kernel
template <class S, bool BF16>
__global__ void __launch_bounds__(S::THREADS, S::MINB)
grad_rows_kernel(const __grid_constant__ Maps maps, const GradParams p) {
  constexpr int NT = S::NT, HD = S::HD, CG = S::CG, PITCH = S::PITCH, STAGES = S::STAGES;
  using R = Rows<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* red = reinterpret_cast<float*>(smem + STAGES * S::STAGE);       // [2][warp][16][PITCH]
  float4* ex = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(red) + S::RED);  // [2][CG][64]
  uint32_t* mask_s = reinterpret_cast<uint32_t*>(ex + 2 * CG * kBR);     // [NPAD][4]
  Tail* tail = reinterpret_cast<Tail*>(mask_s + S::NPAD * 4);

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
  const uint32_t warps = uint32_t((rows + 15) / 16 * CG);  // live ones
  const int count = (p.B - share + p.S - 1) / p.S;
  const int i0 = row0 + rg * 16 + g, i1 = i0 + 8;  // this thread's two query rows
  const int jb = cg * S::WC + 2 * t4;              // its first column; tile t adds 8 t
  const float c1 = p.scale * kLog2e;

  auto issue = [&](int k) {
    const int st = k % STAGES, b = share + k * p.S;
    uint8_t* base = smem + st * S::STAGE;
    uint64_t* full = &tail->full[st];
    if (p.analytic) tail->last[st] = last_axes(p, b);
    tail->issued = k + 1;
    mbar_arrive_expect_tx(full, S::STAGE);
    load_rows<HD, S::NPAD>(base, &maps.cols0, full, 0, h, b);
    load_rows<HD, S::NPAD>(base + S::COLS, &maps.cols1, full, 0, h, b);
    load_rows<HD, kBR>(base + 2 * S::COLS, &maps.rows0, full, row0, h, b);
    load_rows<HD, kBR>(base + 2 * S::COLS + S::ROWS, &maps.rows1, full, row0, h, b);
  };
  if (tid == 0) {
    init_tail(tail);
    for (int k = 0; k < STAGES && k < count; ++k) issue(k);
  }
  uint32_t code0 = 0, code1 = 0;
  const uint32_t pen = p.mask_pen;
  if (p.analytic) {
    for (int i = tid; i < S::NPAD * 4; i += S::THREADS)
      mask_s[i] = i / 4 < p.N ? col_feature(p.mask_one, side_code(p, i / 4), i % 4) : 0u;
    code0 = i0 < p.N ? side_code(p, i0) : 0u;
    code1 = i1 < p.N ? side_code(p, i1) : 0u;
  }
  if (warp == 0) {
    tmem_alloc(&tail->tm_slot, S::TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // a warp reads and writes the 32 tensor-memory lanes of its quarter
  const uint32_t tm =
      tail->tm_slot + (uint32_t(32 * (warp & 3)) << 16) + uint32_t((warp >> 2) * S::WC);
  const uint32_t tm_bias = tm, tm_sum = tm + NT * 4;

  if (live) {
    {
      float v[NT][4];
      start_values<NT, BF16, false>(p, h, i0, jb, v);
      tm_st<NT * 4>(tm_bias, v[0]);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[t][e] = 0.f;
      tm_st<NT * 4>(tm_sum, v[0]);
      tmem_wait_st();
    }
    const int width = p.H * HD, tok = 3 * width;  // elements per token of the output and of qkv
    // dq of window k: the sum of the CG warps' parts
    auto join = [&](int k) {
      const float* all = red + ((k & 1) * S::WARPS + rg * CG) * 16 * PITCH;
      uint16_t* to = p.dqkv + ((long long)(share + k * p.S) * p.N + row0 + rg * 16) * tok + h * HD;
#pragma unroll
      for (int o = cg * 32 + lane; o < 16 * HD / 2; o += 32 * CG) {
        const int r = o / (HD / 2), c = (o % (HD / 2)) * 2;
        float2 v = *reinterpret_cast<const float2*>(all + r * PITCH + c);
#pragma unroll
        for (int w = 1; w < CG; ++w)
          v = __fadd2_rn(v, *reinterpret_cast<const float2*>(all + (w * 16 + r) * PITCH + c));
        if (row0 + rg * 16 + r < p.N)
          *reinterpret_cast<uint32_t*>(to + r * tok + c) = pack2<BF16>(v.x, v.y);
      }
    };

    // lane parts of the ldmatrix addresses
    const uint32_t a_off = R::at(rg * 16 + (lane & 15), lane >> 4);
    const uint32_t a_off1 = HD == 32 ? R::at(rg * 16 + (lane & 15), (lane >> 4) + 2) : 0u;
    const uint32_t col0 = uint32_t(cg * S::WC * R::BYTES);
    const uint32_t b_off =
        col0 + (HD == 16 ? R::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1)  // 2 tiles
                         : R::at(lane & 7, lane >> 3));                          // 1 tile
    const uint32_t bt_off = col0 + R::at(lane & 15, lane >> 4);
    const uint32_t bt_off1 = HD == 32 ? col0 + R::at(lane & 15, (lane >> 4) + 2) : 0u;

#pragma unroll 1
    for (int k = 0; k < count; ++k) {
      // scores: the accumulators start at bias / scale
      float s[NT][4];
      wait_stage<STAGES>(tail, k);
      tm_ld<NT * 4>(tm_bias, s[0]);
      const uint32_t ks = smem_u32(smem) + uint32_t((k % STAGES) * S::STAGE);
      const uint32_t vs = ks + S::COLS, qs = vs + S::COLS, gs = qs + S::ROWS;
      {
        uint32_t a[R::KS][4];
        ldsm_x4(qs + a_off, a[0]);
        if constexpr (HD == 32) ldsm_x4(qs + a_off1, a[1]);
        tm_wait<NT>(s);
        if constexpr (HD == 16) {
#pragma unroll
          for (int t = 0; t < NT; t += 2) {
            uint32_t bf[4];  // past the last tile: rows of the next warp, V or Q, not used
            ldsm_x4(ks + b_off + uint32_t(8 * t * R::BYTES), bf);
            mma16<BF16>(s[t], a[0], bf[0], bf[1], s[t]);
            if (t + 1 < NT) mma16<BF16>(s[t + 1], a[0], bf[2], bf[3], s[t + 1]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            uint32_t bf[4];
            ldsm_x4(ks + b_off + uint32_t(8 * t * R::BYTES), bf);
            mma16<BF16>(s[t], a[0], bf[0], bf[1], s[t]);
            mma16<BF16>(s[t], a[1], bf[2], bf[3], s[t]);
          }
        }
      }
      float g0 = 1.f, g1 = 1.f;
      uint32_t ga[R::KS][4];
      ldsm_x4(gs + a_off, ga[0]);
      if constexpr (HD == 32) ldsm_x4(gs + a_off1, ga[1]);
      if constexpr (!BF16) {  // power-of-two scale of ds, from the row's largest |do|
        __half2 h0 = __float2half2_rn(0.f), h1 = h0;
#pragma unroll
        for (int q = 0; q < R::KS; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 v = __habs2(*reinterpret_cast<const __half2*>(&ga[q][e]));
            if (e & 1) h1 = __hmax2(h1, v);
            else h0 = __hmax2(h0, v);
          }
        float am0 = __half2float(__hmax(__low2half(h0), __high2half(h0)));
        float am1 = __half2float(__hmax(__low2half(h1), __high2half(h1)));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          am0 = fmaxf(am0, __shfl_xor_sync(~0u, am0, o));
          am1 = fmaxf(am1, __shfl_xor_sync(~0u, am1, o));
        }
        g0 = grad_scale(am0);
        g1 = grad_scale(am1);
        if (cg == 0) {  // the row group's, for the columns kernel
          am0 = fmaxf(am0, am1);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) am0 = fmaxf(am0, __shfl_xor_sync(~0u, am0, o));
          if (lane == 0)
            p.amax[((long long)(share + k * p.S) * p.H + h) * ((p.N + 15) / 16) + rb * kRG + rg] =
                am0;
        }
      }
      // dp = do v^T of a pair of tiles, taken twice: for its sum with p, and again for ds once the
      // row's statistics are known.  Keeping it instead (44 registers more) left the scheduler
      // nothing to overlap with.
      float d[2][2][4];
      auto dp_pair = [&](int t) {
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        float(&dd)[2][4] = d[(t >> 1) & 1];
        if constexpr (HD == 16) {
          uint32_t bf[4];  // past the last tile: rows of the next warp or of Q, not used
          ldsm_x4(vs + b_off + uint32_t(8 * t * R::BYTES), bf);
          mma16<BF16>(dd[0], ga[0], bf[0], bf[1], z);
          if (t + 1 < NT) mma16<BF16>(dd[1], ga[0], bf[2], bf[3], z);
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (t + u >= NT) break;
            uint32_t bf[4];
            ldsm_x4(vs + b_off + uint32_t(8 * (t + u) * R::BYTES), bf);
            mma16<BF16>(dd[u], ga[0], bf[0], bf[1], z);
            mma16<BF16>(dd[u], ga[1], bf[2], bf[3], dd[u]);
          }
        }
      };
      dp_pair(0);
      if (p.analytic) {
        const uint32_t last = tail->last[k % STAGES];
        if (last != 0) {
          const uint32_t a0 = row_feature(pen, code0, last, t4), a1 = row_feature(pen, code1, last, t4);
          const uint32_t* mb = mask_s + (cg * S::WC + g) * 4 + t4;
#pragma unroll
          for (int t = 0; t < NT; ++t) mma8<BF16>(s[t], a0, a1, mb[32 * t]);
        }
      }
      // maxima of this warp's columns (a warp of padded columns only: a finite stand-in)
      float m0 = -1e30f, m1 = -1e30f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        m0 = max3(m0, s[t][0], s[t][1]);
        m1 = max3(m1, s[t][2], s[t][3]);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(~0u, m0, o));
        m1 = fmaxf(m1, __shfl_xor_sync(~0u, m1, o));
      }
      const float2 cc = both(c1), n0 = both(-m0 * c1), n1 = both(-m1 * c1);
      float2 l0 = both(0.f), l1 = both(0.f);  // sums of exponentials
      float2 e0 = both(0.f), e1 = both(0.f);  // sums of p dp
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t % 2 == 0 && t + 2 < NT) dp_pair(t + 2);
        const float(&dt)[4] = d[(t >> 1) & 1][t & 1];
        const float2 x0 = __ffma2_rn(two(s[t], 0), cc, n0), x1 = __ffma2_rn(two(s[t], 1), cc, n1);
        const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y)), p1 = make_float2(ex2(x1.x), ex2(x1.y));
        l0 = __fadd2_rn(l0, p0);
        l1 = __fadd2_rn(l1, p1);
        e0 = __ffma2_rn(p0, two(dt, 0), e0);
        e1 = __ffma2_rn(p1, two(dt, 1), e1);
        put(s[t], 0, p0);
        put(s[t], 1, p1);
      }
      // (sum of exponentials, sum of p dp) of the two rows
      float2 q0 = make_float2(l0.x + l0.y, e0.x + e0.y), q1 = make_float2(l1.x + l1.y, e1.x + e1.y);
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        q0 = __fadd2_rn(q0, make_float2(__shfl_xor_sync(~0u, q0.x, o), __shfl_xor_sync(~0u, q0.y, o)));
        q1 = __fadd2_rn(q1, make_float2(__shfl_xor_sync(~0u, q1.x, o), __shfl_xor_sync(~0u, q1.y, o)));
      }
      dp_pair(0);       // for ds, while the row's warps meet
      tmem_wait_st();   // the previous window's dbias is written
      float r0 = 1.f, r1 = 1.f;  // this warp's exponentials relative to the row's
      if constexpr (CG > 1) {
        float4* x = ex + (k & 1) * CG * kBR + rg * 16;
        if (t4 == 0) {
          x[cg * kBR + g] = make_float4(m0, q0.x, q0.y, 0.f);
          x[cg * kBR + g + 8] = make_float4(m1, q1.x, q1.y, 0.f);
        }
        bar_sync(1 + rg, 32 * CG);
        if (k > 0) join(k - 1);
        // every warp of the row adds the same parts in the same order
        const float own0 = m0, own1 = m1;
        float4 y0[CG], y1[CG];
#pragma unroll
        for (int c = 0; c < CG; ++c) {
          y0[c] = x[c * kBR + g];
          y1[c] = x[c * kBR + g + 8];
          m0 = fmaxf(m0, y0[c].x);
          m1 = fmaxf(m1, y1[c].x);
        }
        q0 = q1 = both(0.f);
#pragma unroll
        for (int c = 0; c < CG; ++c) {
          q0 = __ffma2_rn(make_float2(y0[c].y, y0[c].z), both(ex2((y0[c].x - m0) * c1)), q0);
          q1 = __ffma2_rn(make_float2(y1[c].y, y1[c].z), both(ex2((y1[c].x - m1) * c1)), q1);
        }
        r0 = ex2((own0 - m0) * c1);
        r1 = ex2((own1 - m1) * c1);
      } else {
        __syncwarp();
        if (k > 0) join(k - 1);
      }
      const float inv0 = rcp(q0.x), inv1 = rcp(q1.x);
      const float del0 = q0.y * inv0, del1 = q1.y * inv1;
      if (cg == 0 && t4 == 0) {  // statistics for the columns kernel
        float* to = p.stats + ((long long)(share + k * p.S) * p.H + h) * p.NS * 2;
        auto keep = [&](int i, float m, float2 q, float del) {
          if (i >= p.NS) return;
          // (row N of an odd N is copied along by the columns kernel: its p has to be finite)
          to[(i >> 1) * 4 + (i & 1)] = i < p.N ? -fmaf(m, c1, __log2f(q.x)) : 0.f;
          to[(i >> 1) * 4 + (i & 1) + 2] = i < p.N ? -del : 0.f;
        };
        keep(i0, m0, q0, del0);
        keep(i1, m1, q1, del1);
      }
      // ds = p (dp - delta), times the row's power of two in fp16; dbias += ds; dq += ds k with ds
      // rounded to the element type: the rounding errors of a row's keys are independent, so they
      // add up like one rounding of dq itself
      const float2 v0 = both(r0 * inv0 * g0), v1 = both(r1 * inv1 * g1);
      const float2 w0 = both(-del0 * v0.x), w1 = both(-del1 * v1.x);
      const float u0 = inverse_scale(g0), u1 = inverse_scale(g1);
      float acc[HD / 8][4];
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll
      for (int t = 0; t < NT; t += 2) {
        constexpr int kLast = NT - 1;
        const bool pair = t < kLast;
        float sum[2][4];
        if (pair) tm_ld<8>(tm_sum + 4 * t, sum[0]);
        else tm_ld<4>(tm_sum + 4 * t, sum[0]);
        uint32_t bf[HD / 16][4];  // past the last tile: as above
#pragma unroll
        for (int n = 0; n < HD / 16; ++n)
          ldsm_x4_t(ks + (n ? bt_off1 : bt_off) + uint32_t(8 * t * R::BYTES), bf[n]);
        if (t + 2 < NT) dp_pair(t + 2);
        float ds[2][4];
        uint32_t a[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (t + u >= NT) break;
          const float(&dt)[4] = d[(t >> 1) & 1][u];
          put(ds[u], 0, __fmul2_rn(two(s[t + u], 0), __ffma2_rn(two(dt, 0), v0, w0)));
          put(ds[u], 1, __fmul2_rn(two(s[t + u], 1), __ffma2_rn(two(dt, 1), v1, w1)));
          a[2 * u] = pack2<BF16>(ds[u][0], ds[u][1]);
          a[2 * u + 1] = pack2<BF16>(ds[u][2], ds[u][3]);
        }
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) {
          if (pair) {
            mma16<BF16>(acc[2 * n], a, bf[n][0], bf[n][1], acc[2 * n]);
            mma16<BF16>(acc[2 * n + 1], a, bf[n][2], bf[n][3], acc[2 * n + 1]);
          } else {
            mma8<BF16>(acc[2 * n], a[0], a[1], bf[n][0]);
            mma8<BF16>(acc[2 * n + 1], a[0], a[1], bf[n][2]);
          }
        }
        if (pair) tm_wait<2>(sum);
        else tm_wait<1>(reinterpret_cast<float(&)[1][4]>(sum));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (t + u >= NT) break;
          if constexpr (BF16) {
            put(sum[u], 0, __fadd2_rn(two(sum[u], 0), two(ds[u], 0)));
            put(sum[u], 1, __fadd2_rn(two(sum[u], 1), two(ds[u], 1)));
          } else {
            put(sum[u], 0, __ffma2_rn(two(ds[u], 0), both(u0), two(sum[u], 0)));
            put(sum[u], 1, __ffma2_rn(two(ds[u], 1), both(u1), two(sum[u], 1)));
          }
        }
        if (pair) tm_st<8>(tm_sum + 4 * t, sum[0]);
        else tm_st<4>(tm_sum + 4 * t, sum[0]);
      }
      if (release_stage<STAGES>(tail, k, count, warps)) issue(k + STAGES);
      // this warp's part of dq, joined behind the next window's barrier
      const float h0 = p.scale * u0, h1 = p.scale * u1;
      float* mine = red + ((k & 1) * S::WARPS + warp) * 16 * PITCH + g * PITCH + 2 * t4;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        *reinterpret_cast<float2*>(mine + 8 * n) = make_float2(acc[n][0] * h0, acc[n][1] * h0);
        *reinterpret_cast<float2*>(mine + 8 * PITCH + 8 * n) =
            make_float2(acc[n][2] * h1, acc[n][3] * h1);
      }
    }
    if (count > 0) {
      bar_sync(1 + rg, 32 * CG);
      join(count - 1);
    }
    // the head's dbias of this share of the windows
    tmem_wait_st();
    float* out = p.dbias + ((long long)share * p.H + h) * p.N * p.N;
    float v[NT][4];
    tm_ld<NT * 4>(tm_sum, v[0]);
    tm_wait<NT>(v);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = e < 2 ? i0 : i1, j = jb + 8 * t + (e & 1);
        if (i < p.N && j < p.N) out[(long long)i * p.N + j] = v[t][e];
      }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) finish_ring<STAGES>(tail);
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tail->tm_slot, S::TM_COLS);
  }
}

// --------------------------------------------------------------------- columns kernel
// A warp's rows are 16 keys, its columns all queries: p and ds come from the statistics, are
// rounded and multiplied by do and q at once, two tiles of 8 queries at a time.
template <class S, bool BF16>
__global__ void __launch_bounds__(S::THREADS, S::MINB)
grad_cols_kernel(const __grid_constant__ Maps maps, const GradParams p) {
  constexpr int NT = S::NT, HD = S::HD, STAGES = S::STAGES, TT = S::TT;
  using R = Rows<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint32_t* mask_s = reinterpret_cast<uint32_t*>(smem + STAGES * S::STAGE);  // [NPAD][4]
  Tail* tail = reinterpret_cast<Tail*>(mask_s + S::NPAD * 4);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  int blk = blockIdx.x;
  const int share = blk % p.S;
  blk /= p.S;
  const int rb = blk % p.RB, h = blk / p.RB;
  const int row0 = rb * S::BR;
  const int rows = min(S::BR, p.N - row0);
  const bool live = warp * 16 < rows;
  const uint32_t warps = uint32_t((rows + 15) / 16);
  const int count = (p.B - share + p.S - 1) / p.S;
  const int k0 = row0 + warp * 16 + g, k1 = k0 + 8;  // this thread's two keys
  const int groups = (p.N + 15) / 16;
  const uint32_t stat_bytes = uint32_t(p.NS) * 8u;

  auto issue = [&](int k) {
    const int st = k % STAGES, b = share + k * p.S;
    uint8_t* base = smem + st * S::STAGE;
    uint64_t* full = &tail->full[st];
    if (p.analytic) tail->last[st] = last_axes(p, b);
    tail->issued = k + 1;
    mbar_arrive_expect_tx(full, 2 * S::COLS + 2 * S::ROWS + stat_bytes);
    load_rows<HD, S::NPAD>(base, &maps.cols0, full, 0, h, b);
    load_rows<HD, S::NPAD>(base + S::COLS, &maps.cols1, full, 0, h, b);
    load_rows<HD, S::BR>(base + 2 * S::COLS, &maps.rows0, full, row0, h, b);
    load_rows<HD, S::BR>(base + 2 * S::COLS + S::ROWS, &maps.rows1, full, row0, h, b);
    bulk_load(base + 2 * S::COLS + 2 * S::ROWS, p.stats + ((long long)b * p.H + h) * p.NS * 2,
              stat_bytes, full);
  };
  // the statistics of padded queries are not copied: 0 (read as p = 2^-inf)
  for (int i = tid; i < STAGES * S::NPAD; i += S::THREADS)
    *reinterpret_cast<float2*>(smem + (i / S::NPAD) * S::STAGE + 2 * S::COLS + 2 * S::ROWS +
                               (i % S::NPAD) * 8) = make_float2(0.f, 0.f);
  uint32_t code0 = 0, code1 = 0;
  const uint32_t pen = p.mask_pen;
  if (p.analytic) {
    for (int i = tid; i < S::NPAD * 4; i += S::THREADS)
      mask_s[i] = i / 4 < p.N ? col_feature(p.mask_one, side_code(p, i / 4), i % 4) : 0u;
    code0 = k0 < p.N ? side_code(p, k0) : 0u;
    code1 = k1 < p.N ? side_code(p, k1) : 0u;
  }
  if (warp == 0) {
    tmem_alloc(&tail->tm_slot, S::TM_COLS);
    tmem_relinquish();
  }
  if (tid == 0) init_tail(tail);
  fence_proxy_async_shared();  // the zeroed statistics, before the copies over them
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0)
    for (int k = 0; k < STAGES && k < count; ++k) issue(k);
  const uint32_t tm_bias =
      tail->tm_slot + (uint32_t(32 * (warp & 3)) << 16) + uint32_t((warp >> 2) * 4 * TT);

  if (live) {
    float rest[2][4];  // the start values of the tiles past TT
    {
      constexpr int PART = TT == 42 ? 14 : TT == 28 ? 7 : 8;  // tiles per round of gathers
      static_assert(TT % PART == 0, "whole rounds");
#pragma unroll 1
      for (int t = 0; t < TT; t += PART) {
        float v[PART][4];
        start_values<PART, BF16, true>(p, h, k0, 8 * t + 2 * t4, v);
        tm_st<4 * PART>(tm_bias + 4 * t, v[0]);
      }
      if constexpr (TT < NT) start_values<2, BF16, true>(p, h, k0, 8 * TT + 2 * t4, rest);
      tmem_wait_st();
    }
    const int width = p.H * HD, tok = 3 * width;
    const float2 cc = both(p.scale * kLog2e);
    const uint32_t a_off = R::at(warp * 16 + (lane & 15), lane >> 4);
    const uint32_t a_off1 = HD == 32 ? R::at(warp * 16 + (lane & 15), (lane >> 4) + 2) : 0u;
    const uint32_t b_off = HD == 16 ? R::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1)
                                    : R::at(lane & 7, lane >> 3);
    const uint32_t bt_off = R::at(lane & 15, lane >> 4);
    const uint32_t bt_off1 = HD == 32 ? R::at(lane & 15, (lane >> 4) + 2) : 0u;
    const float* amax = p.amax + ((long long)share * p.H + h) * groups + lane;
    const long long amax_step = (long long)p.S * p.H * groups;
    float am = 0.f;  // the next window's, fetched one window ahead
    if constexpr (!BF16) am = lane < groups ? __ldg(amax) : 0.f;

#pragma unroll 1
    for (int k = 0; k < count; ++k) {
      // one power-of-two scale of ds for the window (fp16): its sum over the queries goes
      // through one accumulator
      float gscale = 1.f;
      if constexpr (!BF16) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(~0u, am, o));
        gscale = grad_scale(am);
        am = lane < groups && k + 1 < count ? __ldg(amax + (k + 1) * amax_step) : 0.f;
      }
      float nb[2][4];  // start values of the next pair of tiles
      wait_stage<STAGES>(tail, k);
      tm_ld<8>(tm_bias, nb[0]);
      const uint32_t qs = smem_u32(smem) + uint32_t((k % STAGES) * S::STAGE);
      const uint32_t gs = qs + S::COLS, ks = gs + S::COLS, vs = ks + S::ROWS;
      const float2* stat = reinterpret_cast<const float2*>(
          smem + (k % STAGES) * S::STAGE + 2 * S::COLS + 2 * S::ROWS) + 2 * t4;
      uint32_t last = 0;
      if (p.analytic) last = tail->last[k % STAGES];
      const uint32_t a0 = row_feature(pen, code0, last, t4), a1 = row_feature(pen, code1, last, t4);
      const uint32_t* mb = mask_s + g * 4 + t4;

      uint32_t ka[R::KS][4], va[R::KS][4];
      ldsm_x4(ks + a_off, ka[0]);
      ldsm_x4(vs + a_off, va[0]);
      if constexpr (HD == 32) {
        ldsm_x4(ks + a_off1, ka[1]);
        ldsm_x4(vs + a_off1, va[1]);
      }
      float dk[HD / 8][4], dv[HD / 8][4];
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;

      // The scores and dp of a pair of tiles, one pair ahead of what is made of them
      float s[2][2][4], d[2][2][4];
      auto products = [&](auto masked, int t) {
        constexpr float z[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t at = uint32_t(8 * t * R::BYTES);
        float(&sp)[2][4] = s[(t >> 1) & 1];
        float(&dp)[2][4] = d[(t >> 1) & 1];
        if (t < TT) tm_wait<2>(nb);
        if constexpr (HD == 16) {
          uint32_t bq[4], bg[4];
          ldsm_x4(qs + b_off + at, bq);
          ldsm_x4(gs + b_off + at, bg);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            mma16<BF16>(sp[u], ka[0], bq[2 * u], bq[2 * u + 1], t < TT ? nb[u] : rest[u]);
            mma16<BF16>(dp[u], va[0], bg[2 * u], bg[2 * u + 1], z);
          }
        } else {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t bq[4], bg[4];
            ldsm_x4(qs + b_off + at + uint32_t(8 * u * R::BYTES), bq);
            ldsm_x4(gs + b_off + at + uint32_t(8 * u * R::BYTES), bg);
            mma16<BF16>(sp[u], ka[0], bq[0], bq[1], t < TT ? nb[u] : rest[u]);
            mma16<BF16>(dp[u], va[0], bg[0], bg[1], z);
            mma16<BF16>(sp[u], ka[1], bq[2], bq[3], sp[u]);
            mma16<BF16>(dp[u], va[1], bg[2], bg[3], dp[u]);
          }
        }
        if (t + 2 < TT) tm_ld<8>(tm_bias + 4 * (t + 2), nb[0]);
        if constexpr (decltype(masked)::value) {
#pragma unroll
          for (int u = 0; u < 2; ++u) mma8<BF16>(sp[u], a0, a1, mb[32 * (t + u)]);
        }
      };
      auto sweep = [&](auto masked) {
        products(masked, 0);
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          const uint32_t at = uint32_t(8 * t * R::BYTES);
          uint32_t tq[HD / 16][4], tg[HD / 16][4];
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            ldsm_x4_t(gs + (n ? bt_off1 : bt_off) + at, tg[n]);
            ldsm_x4_t(qs + (n ? bt_off1 : bt_off) + at, tq[n]);
          }
          if (t + 2 < NT) products(masked, t + 2);
          uint32_t pa[4], da[4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // two queries' statistics: (-lse, -lse, -delta, -delta)
            const float4 x = *reinterpret_cast<const float4*>(stat + 8 * (t + u));
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float2 y =
                  __ffma2_rn(two(s[(t >> 1) & 1][u], r), cc, make_float2(x.x, x.y));
              const float2 q = make_float2(ex2(y.x), ex2(y.y));
              float2 ds = __fmul2_rn(
                  __fadd2_rn(two(d[(t >> 1) & 1][u], r), make_float2(x.z, x.w)), q);
              if constexpr (!BF16) ds = __fmul2_rn(ds, both(gscale));
              pa[2 * u + r] = pack2<BF16>(q.x, q.y);
              da[2 * u + r] = pack2<BF16>(ds.x, ds.y);
            }
          }
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            mma16<BF16>(dv[2 * n], pa, tg[n][0], tg[n][1], dv[2 * n]);
            mma16<BF16>(dv[2 * n + 1], pa, tg[n][2], tg[n][3], dv[2 * n + 1]);
            mma16<BF16>(dk[2 * n], da, tq[n][0], tq[n][1], dk[2 * n]);
            mma16<BF16>(dk[2 * n + 1], da, tq[n][2], tq[n][3], dk[2 * n + 1]);
          }
        }
      };
      if (last != 0) sweep(std::true_type{});
      else sweep(std::false_type{});
      if (release_stage<STAGES>(tail, k, count, warps)) issue(k + STAGES);
      const float f = BF16 ? p.scale : p.scale * inverse_scale(gscale);
      uint16_t* to = p.dqkv + ((long long)(share + k * p.S) * p.N + k0) * tok + width + h * HD + 2 * t4;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        if (k0 < p.N) {
          *reinterpret_cast<uint32_t*>(to + 8 * n) = pack2<BF16>(dk[n][0] * f, dk[n][1] * f);
          *reinterpret_cast<uint32_t*>(to + width + 8 * n) = pack2<BF16>(dv[n][0], dv[n][1]);
        }
        if (k1 < p.N) {
          *reinterpret_cast<uint32_t*>(to + 8 * tok + 8 * n) = pack2<BF16>(dk[n][2] * f, dk[n][3] * f);
          *reinterpret_cast<uint32_t*>(to + 8 * tok + width + 8 * n) = pack2<BF16>(dv[n][2], dv[n][3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0) finish_ring<STAGES>(tail);
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tail->tm_slot, S::TM_COLS);
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// 4D map {head_dim, N, H, B} over one part of the tokens (`tok` elements per token), in boxes of
// `rows` rows; rows past N are zero-filled.
int make_map(CUtensorMap* map, const void* base, const AttnGradArgs& a, int64_t tok, int rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return set_error(kErrCuda, "cuTensorMapEncodeTiled is unavailable");
  const cuuint64_t dims[4] = {cuuint64_t(a.head_dim), cuuint64_t(a.N), cuuint64_t(a.H),
                              cuuint64_t(a.B)};
  const cuuint64_t strides[3] = {cuuint64_t(tok) * 2, cuuint64_t(a.head_dim) * 2,
                                 cuuint64_t(tok) * cuuint64_t(a.N) * 2};
  const cuuint32_t box[4] = {cuuint32_t(a.head_dim), cuuint32_t(rows), 1u, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUresult r = enc(
      map, a.dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      a.head_dim == 16 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_64B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(kErrInvalid, "cuTensorMapEncodeTiled rejected a tensor");
  return kOk;
}

int make_maps(Maps* m, const AttnGradArgs& a, bool of_rows_kernel, int cols, int rows) {
  const int64_t width = a.H * a.head_dim;
  const uint16_t* q = static_cast<const uint16_t*>(a.qkv);
  CUtensorMap* const qo[2] = {of_rows_kernel ? &m->rows0 : &m->cols0,
                              of_rows_kernel ? &m->rows1 : &m->cols1};
  CUtensorMap* const kv[2] = {of_rows_kernel ? &m->cols0 : &m->rows0,
                              of_rows_kernel ? &m->cols1 : &m->rows1};
  const int qo_box = box_rows(of_rows_kernel ? rows : cols);
  const int kv_box = box_rows(of_rows_kernel ? cols : rows);
  if (int e = make_map(qo[0], q, a, 3 * width, qo_box)) return e;
  if (int e = make_map(qo[1], a.grad_out, a, width, qo_box)) return e;
  if (int e = make_map(kv[0], q + width, a, 3 * width, kv_box)) return e;
  return make_map(kv[1], q + 2 * width, a, 3 * width, kv_box);
}

// parts[0][i] = sum over s of parts[s][i]: 64 elements per CTA, four threads each taking a quarter
// of the parts (8 loads in flight), joined in a fixed order.
__global__ void __launch_bounds__(256) sum_shares_kernel(float* parts, int shares, long long n) {
  __shared__ float quarter[3][64];
  const int x = threadIdx.x & 63, q = threadIdx.x >> 6;
  const long long i = blockIdx.x * 64LL + x;
  float sum = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int s = q; s < shares; s += 4) sum += parts[s * n + i];
  }
  if (q > 0) quarter[q - 1][x] = sum;
  __syncthreads();
  if (q == 0 && i < n) parts[i] = sum + quarter[0][x] + quarter[1][x] + quarter[2][x];
}

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 148;
}

template <class K>
int set_smem(K kernel, int bytes) {
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention gradient smem attribute");
}

// Row blocks and shares of a kernel with `rows` rows per CTA and `per_sm` CTAs per SM: as many
// shares as keep the SMs' CTA slots busy with one CTA per (head, row block, share), at most one
// per window.
void split(GradParams* p, int rows, int per_sm) {
  p->RB = (p->N + rows - 1) / rows;
  const int64_t s = int64_t(sm_count()) * per_sm / (int64_t(p->H) * p->RB);
  p->S = int(s < 1 ? 1 : s > p->B ? p->B : s);
}

template <int NPAD, int HD, bool BF16>
int launch_grad(GradParams p, const AttnGradArgs& a, cudaStream_t stream) {
  using RS = RowsShape<NPAD, HD>;
  using CS = ColsShape<NPAD, HD>;
  static bool configured[64] = {false};  // per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !configured[dev]) {
    if (int e = set_smem(grad_rows_kernel<RS, BF16>, RS::SMEM)) return e;
    if (int e = set_smem(grad_cols_kernel<CS, BF16>, CS::SMEM)) return e;
    if (dev < 64) configured[dev] = true;
  }
  Maps maps;
  if (int e = make_maps(&maps, a, true, NPAD, kBR)) return e;
  p.RB = (p.N + kBR - 1) / kBR;
  p.S = int(a.shares);
  grad_rows_kernel<RS, BF16>
      <<<unsigned(p.H) * unsigned(p.RB) * unsigned(p.S), RS::THREADS, RS::SMEM, stream>>>(maps, p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "attention gradient (rows) launch");
  if (int r = make_maps(&maps, a, false, NPAD, CS::BR)) return r;
  split(&p, CS::BR, CS::MINB);
  grad_cols_kernel<CS, BF16>
      <<<unsigned(p.H) * unsigned(p.RB) * unsigned(p.S), CS::THREADS, CS::SMEM, stream>>>(maps, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "attention gradient (columns) launch");
  return kOk;
}

template <int HD, bool BF16>
int dispatch_npad(const GradParams& p, const AttnGradArgs& a, cudaStream_t stream) {
  if (p.N <= 64) return launch_grad<64, HD, BF16>(p, a, stream);
  if (p.N <= 128) return launch_grad<128, HD, BF16>(p, a, stream);
  if (p.N <= 224) return launch_grad<224, HD, BF16>(p, a, stream);
  return launch_grad<352, HD, BF16>(p, a, stream);
}

}  // namespace

// (H: a window's offsets fit 32 bits)
bool attention_grad_tensor_path(int dtype, int64_t H, int64_t N, int64_t head_dim) {
  return dtype != kF32 && (head_dim == 16 || head_dim == 32) && N >= 1 && N <= 352 && H <= 4096;
}

// Shares of the windows of the rows kernel, each with its own part of the bias gradient.
int64_t attention_grad_shares(int64_t B, int64_t H, int64_t N) {
  GradParams p{};
  p.B = int(B > 0 ? B : 1);
  p.H = int(H);
  p.N = int(N);
  split(&p, kBR, N <= 64 ? 4 : N <= 128 ? 2 : 1);  // RowsShape::MINB
  return p.S;
}

int launch_sum_shares(float* parts, int64_t shares, int64_t n, cudaStream_t stream) {
  if (shares <= 1 || n == 0) return kOk;
  sum_shares_kernel<<<unsigned((n + 63) / 64), 256, 0, stream>>>(parts, int(shares), n);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? kOk : set_cuda_error(e, "attention gradient sum launch");
}

int read_attention_grad_error(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_grad_error, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_grad_error, &zero, sizeof(int));
  }
  return v;
}

int training_error_word(int** word) {
  static std::mutex mu;
  static void* at[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  void* p = e == cudaSuccess && dev < 64 ? at[dev] : nullptr;
  if (e == cudaSuccess && p == nullptr) e = cudaGetSymbolAddress(&p, g_grad_error);
  if (e != cudaSuccess) return set_cuda_error(e, "error word of the training kernels");
  if (dev < 64) at[dev] = p;
  *word = static_cast<int*>(p);
  return kOk;
}

int launch_attention_grad(const AttnGradArgs& a, cudaStream_t stream) {
  GradParams p{};
  p.dqkv = static_cast<uint16_t*>(a.grad_qkv);
  p.dbias = a.grad_bias;
  p.stats = a.stats;
  p.NS = int(a.N + (a.N & 1));
  p.amax = a.stats + 2 * a.B * a.H * p.NS;
  p.table = a.table;
  p.pairs = a.pairs;
  p.table_f32 = a.table_f32 ? 1 : 0;
  p.table_rows = int(a.table_rows);
  p.analytic = (a.shift[0] | a.shift[1] | a.shift[2]) != 0;
  if (p.analytic) {
    const MaskPenalty m = mask_penalty(a.scale, a.dtype == kBF16);
    p.mask_pen = m.pen;
    p.mask_one = m.one;
  }
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
  p.scale = a.scale;
  const bool bf16 = a.dtype == kBF16;
  if (a.head_dim == 32)
    return bf16 ? dispatch_npad<32, true>(p, a, stream) : dispatch_npad<32, false>(p, a, stream);
  return bf16 ? dispatch_npad<16, true>(p, a, stream) : dispatch_npad<16, false>(p, a, stream);
}

}  // namespace crumpet
