// crumpet_b200: the C ABI (declared in include/crumpet_b200.h).
//
// Every entry point validates its arguments the way the reference's Python
// wrappers and C++ ops do (torch-ext/crumpet/__init__.py:89-123,
// cuda/attn_mask_3d.cu:143), launches on the caller's stream, never allocates
// and never synchronises.  Failures return a non-zero status and leave a
// message for crumpet_last_error().
#include <cmath>
#include <cstdio>
#include <cstring>

#include "../../include/crumpet_b200.h"
#include "common.cuh"
#include "kernels.h"

namespace crumpet {

static_assert(kTensorMinScale == CRUMPET_TENSOR_MIN_SCALE, "as the header says");

namespace {
thread_local char g_last_error[512] = {0};
}

int set_error(int code, const char* msg) {
  std::snprintf(g_last_error, sizeof(g_last_error), "%s", msg);
  return code;
}

int set_cuda_error(cudaError_t err, const char* where) {
  std::snprintf(g_last_error, sizeof(g_last_error), "%s: %s", where, cudaGetErrorString(err));
  return kErrCuda;
}

MaskPenalty mask_penalty(float scale, bool bf16) {
  const auto bits = [&](double v) -> uint32_t {
    return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(float(v)))
                : __half_as_ushort(__float2half_rn(float(v)));
  };
  const auto value = [&](uint32_t b) -> double {
    return bf16 ? __bfloat162float(__ushort_as_bfloat16(uint16_t(b)))
                : __half2float(__ushort_as_half(uint16_t(b)));
  };
  const double want = -100.0 / double(scale);
  MaskPenalty best{bits(want), bits(1.0)};
  double least = std::fabs(value(best.pen) - want);
  for (int i = 1; i < 128 && least > 0.0; ++i) {  // 1 + i / 128: a number of either type
    const double one = 1.0 + i / 128.0;
    const uint32_t pen = bits(want / one);
    const double off = std::fabs(value(pen) * one - want);
    if (off < least) {
      least = off;
      best = MaskPenalty{pen, bits(one)};
    }
  }
  return best;
}

namespace {

int check_dtype(int dtype) {
  if (dtype != kF32 && dtype != kF16 && dtype != kBF16)
    return set_error(kErrInvalid, "CRUMPET supports float32, float16 and bfloat16");
  return kOk;
}

// Mirrors _validate_shape (torch-ext/crumpet/__init__.py:98-117).
int check_window_shape(int64_t D, int64_t H, int64_t W, int64_t ws_d, int64_t ws_h, int64_t ws_w,
                       int64_t ss_d, int64_t ss_h, int64_t ss_w) {
  if (D <= 0 || H <= 0 || W <= 0) return set_error(kErrInvalid, "D, H and W must be positive");
  if (ws_d <= 0 || ws_h <= 0 || ws_w <= 0)
    return set_error(kErrInvalid, "window_size values must be positive");
  if (D % ws_d || H % ws_h || W % ws_w)
    return set_error(kErrInvalid,
                     "standalone CRUMPET kernels require D, H and W to be divisible by window_size");
  const int64_t ss[3] = {ss_d, ss_h, ss_w};
  const int64_t ws[3] = {ws_d, ws_h, ws_w};
  for (int a = 0; a < 3; ++a) {
    if (ss[a] < 0 || ss[a] >= ws[a]) {
      char buf[96];
      std::snprintf(buf, sizeof(buf), "shift_size[%d] must satisfy 0 <= shift < window_size[%d]", a,
                    a);
      return set_error(kErrInvalid, buf);
    }
  }
  // 32-bit index arithmetic inside one window and one volume slice.
  if (D * H * W >= (int64_t(1) << 31)) return set_error(kErrInvalid, "D*H*W must be below 2^31");
  return kOk;
}

int window_copy(bool forward, void* out, const void* in, int dtype, int64_t B, int64_t D, int64_t H,
                int64_t W, int64_t C, int64_t ws_d, int64_t ws_h, int64_t ws_w, int64_t ss_d,
                int64_t ss_h, int64_t ss_w, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_window_shape(D, H, W, ws_d, ws_h, ws_w, ss_d, ss_h, ss_w)) return e;
  if (B < 0 || C < 0) return set_error(kErrInvalid, "B and C must be non-negative");
  if (B == 0 || C == 0) return kOk;  // empty output: nothing to do
  if (out == nullptr || in == nullptr) return set_error(kErrInvalid, "null tensor pointer");
  const ShapeArgs s{B, D, H, W, C, ws_d, ws_h, ws_w, ss_d, ss_h, ss_w};
  return launch_window_copy(forward, out, in, s, dtype, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace crumpet

using namespace crumpet;

extern "C" {

const char* crumpet_last_error(void) { return g_last_error; }

int crumpet_abi_version(void) { return CRUMPET_ABI_VERSION; }

int crumpet_fused_shift_partition_3d(void* output, const void* x, int dtype, int64_t B, int64_t D,
                                     int64_t H, int64_t W, int64_t C, int64_t ws_d, int64_t ws_h,
                                     int64_t ws_w, int64_t ss_d, int64_t ss_h, int64_t ss_w,
                                     void* stream) {
  return window_copy(true, output, x, dtype, B, D, H, W, C, ws_d, ws_h, ws_w, ss_d, ss_h, ss_w,
                     stream);
}

int crumpet_fused_unshift_unpartition_3d(void* output, const void* windows, int dtype, int64_t B,
                                         int64_t D, int64_t H, int64_t W, int64_t C, int64_t ws_d,
                                         int64_t ws_h, int64_t ws_w, int64_t ss_d, int64_t ss_h,
                                         int64_t ss_w, void* stream) {
  return window_copy(false, output, windows, dtype, B, D, H, W, C, ws_d, ws_h, ws_w, ss_d, ss_h,
                     ss_w, stream);
}

int crumpet_fused_shift_partition_3d_backward(void* grad_x, const void* grad_windows, int dtype,
                                              int64_t B, int64_t D, int64_t H, int64_t W,
                                              int64_t C, int64_t ws_d, int64_t ws_h, int64_t ws_w,
                                              int64_t ss_d, int64_t ss_h, int64_t ss_w,
                                              void* stream) {
  return window_copy(false, grad_x, grad_windows, dtype, B, D, H, W, C, ws_d, ws_h, ws_w, ss_d,
                     ss_h, ss_w, stream);
}

int crumpet_fused_unshift_unpartition_3d_backward(void* grad_windows, const void* grad_x,
                                                  int dtype, int64_t B, int64_t D, int64_t H,
                                                  int64_t W, int64_t C, int64_t ws_d, int64_t ws_h,
                                                  int64_t ws_w, int64_t ss_d, int64_t ss_h,
                                                  int64_t ss_w, void* stream) {
  return window_copy(true, grad_windows, grad_x, dtype, B, D, H, W, C, ws_d, ws_h, ws_w, ss_d, ss_h,
                     ss_w, stream);
}

int crumpet_compute_attn_mask_3d(void* output, int dtype, int64_t D, int64_t H, int64_t W,
                                 int64_t ws_d, int64_t ws_h, int64_t ws_w, int64_t ss_d,
                                 int64_t ss_h, int64_t ss_w, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_window_shape(D, H, W, ws_d, ws_h, ws_w, ss_d, ss_h, ss_w)) return e;
  if (output == nullptr) return set_error(kErrInvalid, "null tensor pointer");
  return launch_attn_mask(output, D, H, W, ws_d, ws_h, ws_w, ss_d, ss_h, ss_w, dtype,
                          static_cast<cudaStream_t>(stream));
}

int crumpet_fused_swin_attention(void* out, const void* q, const void* k, const void* v,
                                 const void* rel_bias, const void* mask, int64_t mask_windows,
                                 const uint8_t* boundary, int dtype, int64_t B, int64_t H,
                                 int64_t N, int64_t head_dim, float scale, void* stream) {
  AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.qkv_stride_n = head_dim;
  a.qkv_stride_h = N * head_dim;
  a.qkv_stride_b = H * N * head_dim;
  a.out = out;
  a.out_stride_n = head_dim;
  a.out_stride_h = N * head_dim;
  a.out_stride_b = H * N * head_dim;
  a.bias = rel_bias;
  a.mask = mask;
  a.mask_windows = mask_windows;
  a.boundary = boundary;
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return launch_window_attention(a, static_cast<cudaStream_t>(stream));
}

int crumpet_fused_swin_attention_shifted(void* out, const void* q, const void* k,
                                         const void* v, const void* rel_bias,
                                         const uint8_t* boundary, int dtype, int64_t B,
                                         int64_t H, int64_t N, int64_t head_dim, int64_t nw_d,
                                         int64_t nw_h, int64_t nw_w, int64_t ws_d, int64_t ws_h,
                                         int64_t ws_w, int64_t ss_d, int64_t ss_h, int64_t ss_w,
                                         float scale, void* stream) {
  AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.qkv_stride_n = head_dim;
  a.qkv_stride_h = N * head_dim;
  a.qkv_stride_b = H * N * head_dim;
  a.out = out;
  a.out_stride_n = head_dim;
  a.out_stride_h = N * head_dim;
  a.out_stride_b = H * N * head_dim;
  a.bias = rel_bias;
  a.boundary = boundary;
  a.analytic = (ss_d | ss_h | ss_w) != 0;
  a.nwin[0] = nw_d;
  a.nwin[1] = nw_h;
  a.nwin[2] = nw_w;
  a.win[0] = ws_d;
  a.win[1] = ws_h;
  a.win[2] = ws_w;
  a.shift[0] = ss_d;
  a.shift[1] = ss_h;
  a.shift[2] = ss_w;
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return launch_window_attention(a, static_cast<cudaStream_t>(stream));
}

int crumpet_swin_window_attention_qkv(void* out, const void* qkv, const void* bias_table,
                                      int table_f32, int64_t table_rows, const int64_t* rel_index,
                                      int64_t index_stride, int64_t nw_d, int64_t nw_h,
                                      int64_t nw_w, int64_t ws_d, int64_t ws_h, int64_t ws_w,
                                      int64_t ss_d, int64_t ss_h, int64_t ss_w, int dtype,
                                      int64_t B, int64_t H, int64_t N, int64_t head_dim,
                                      float scale, void* stream) {
  AttnArgs a{};
  const int64_t hd = H * head_dim;
  const int64_t esize = dtype == kF32 ? 4 : 2;
  a.q = qkv;
  a.k = static_cast<const char*>(qkv) + hd * esize;
  a.v = static_cast<const char*>(qkv) + 2 * hd * esize;
  a.qkv_stride_n = 3 * hd;
  a.qkv_stride_h = head_dim;
  a.qkv_stride_b = N * 3 * hd;
  a.out = out;
  a.out_stride_n = hd;
  a.out_stride_h = head_dim;
  a.out_stride_b = N * hd;
  a.bias_from_table = true;
  a.table = bias_table;
  a.table_f32 = table_f32 != 0;
  a.table_rows = table_rows;
  a.index = rel_index;
  a.index_stride = index_stride;
  a.analytic = (ss_d | ss_h | ss_w) != 0;
  a.nwin[0] = nw_d;
  a.nwin[1] = nw_h;
  a.nwin[2] = nw_w;
  a.win[0] = ws_d;
  a.win[1] = ws_h;
  a.win[2] = ws_w;
  a.shift[0] = ss_d;
  a.shift[1] = ss_h;
  a.shift[2] = ss_w;
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return launch_window_attention(a, static_cast<cudaStream_t>(stream));
}

int crumpet_swin_window_attention_qkv_static_tiles(
    void* out, const void* qkv, const void* bias_table, int table_f32, int64_t table_rows,
    const int64_t* rel_index, int64_t index_stride, int64_t nw_d, int64_t nw_h, int64_t nw_w,
    int64_t ws_d, int64_t ws_h, int64_t ws_w, int64_t ss_d, int64_t ss_h, int64_t ss_w,
    int dtype, int64_t B, int64_t H, int64_t N, int64_t head_dim, float scale, void* stream) {
  AttnArgs a{};
  const int64_t hd = H * head_dim;
  const int64_t esize = dtype == kF32 ? 4 : 2;
  a.q = qkv;
  a.k = static_cast<const char*>(qkv) + hd * esize;
  a.v = static_cast<const char*>(qkv) + 2 * hd * esize;
  a.qkv_stride_n = 3 * hd;
  a.qkv_stride_h = head_dim;
  a.qkv_stride_b = N * 3 * hd;
  a.out = out;
  a.out_stride_n = hd;
  a.out_stride_h = head_dim;
  a.out_stride_b = N * hd;
  a.bias_from_table = true;
  a.table = bias_table;
  a.table_f32 = table_f32 != 0;
  a.table_rows = table_rows;
  a.index = rel_index;
  a.index_stride = index_stride;
  a.analytic = (ss_d | ss_h | ss_w) != 0;
  a.nwin[0] = nw_d;
  a.nwin[1] = nw_h;
  a.nwin[2] = nw_w;
  a.win[0] = ws_d;
  a.win[1] = ws_h;
  a.win[2] = ws_w;
  a.shift[0] = ss_d;
  a.shift[1] = ss_h;
  a.shift[2] = ss_w;
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return launch_window_attention_static_tiles(a, static_cast<cudaStream_t>(stream));
}

int64_t crumpet_attention_bias_tiles_bytes(int64_t H, int64_t N) {
  return attention_bias_tiles_bytes(H, N);
}

int crumpet_attention_bias_tiles(void* tiles, const void* bias_table, int table_f32,
                                 int64_t table_rows, const int64_t* rel_index,
                                 int64_t index_stride, int dtype, int64_t H, int64_t N, float scale,
                                 void* stream) {
  AttnArgs a{};
  a.table = bias_table;
  a.table_f32 = table_f32 != 0;
  a.table_rows = table_rows;
  a.index = rel_index;
  a.index_stride = index_stride;
  a.bias_from_table = true;
  a.H = H;
  a.N = N;
  a.scale = scale;
  a.dtype = dtype;
  return launch_attention_bias_tiles(tiles, a, static_cast<cudaStream_t>(stream));
}

int crumpet_swin_window_attention_qkv_tiles(void* out, const void* qkv, const void* bias_tiles,
                                            int64_t nw_d, int64_t nw_h, int64_t nw_w,
                                            int64_t ws_d, int64_t ws_h, int64_t ws_w,
                                            int64_t ss_d, int64_t ss_h, int64_t ss_w, int dtype,
                                            int64_t B, int64_t H, int64_t N, int64_t head_dim,
                                            float scale, void* stream) {
  if (bias_tiles == nullptr) return set_error(kErrInvalid, "null bias tiles");
  AttnArgs a{};
  const int64_t hd = H * head_dim;
  const int64_t esize = dtype == kF32 ? 4 : 2;
  a.q = qkv;
  a.k = static_cast<const char*>(qkv) + hd * esize;
  a.v = static_cast<const char*>(qkv) + 2 * hd * esize;
  a.qkv_stride_n = 3 * hd;
  a.qkv_stride_h = head_dim;
  a.qkv_stride_b = N * 3 * hd;
  a.out = out;
  a.out_stride_n = hd;
  a.out_stride_h = head_dim;
  a.out_stride_b = N * hd;
  a.bias_from_table = true;
  a.bias_tiles = bias_tiles;
  a.analytic = (ss_d | ss_h | ss_w) != 0;
  a.nwin[0] = nw_d;
  a.nwin[1] = nw_h;
  a.nwin[2] = nw_w;
  a.win[0] = ws_d;
  a.win[1] = ws_h;
  a.win[2] = ws_w;
  a.shift[0] = ss_d;
  a.shift[1] = ss_h;
  a.shift[2] = ss_w;
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  return launch_window_attention(a, static_cast<cudaStream_t>(stream));
}

int crumpet_norm_shift_partition_3d(void* output, int out_dtype, const void* x, int in_dtype,
                                    const float* weight, const float* bias, float eps, int64_t B,
                                    int64_t D, int64_t H, int64_t W, int64_t C, int64_t ws_d,
                                    int64_t ws_h, int64_t ws_w, int64_t ss_d, int64_t ss_h,
                                    int64_t ss_w, void* stream) {
  if (int e = check_dtype(out_dtype)) return e;
  if (int e = check_dtype(in_dtype)) return e;
  const int64_t ws[3] = {ws_d, ws_h, ws_w}, ss[3] = {ss_d, ss_h, ss_w};
  return launch_norm_shift_partition(output, out_dtype, x, in_dtype, weight, bias, eps, B, D, H, W,
                                     C, ws, ss, static_cast<cudaStream_t>(stream));
}

int crumpet_unshift_unpartition_crop_3d(void* output, const void* windows, const void* residual,
                                        int dtype, int64_t B, int64_t D, int64_t H, int64_t W,
                                        int64_t C, int64_t ws_d, int64_t ws_h, int64_t ws_w,
                                        int64_t ss_d, int64_t ss_h, int64_t ss_w, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  const int64_t ws[3] = {ws_d, ws_h, ws_w}, ss[3] = {ss_d, ss_h, ss_w};
  return launch_unshift_unpartition_crop(output, windows, residual, dtype, B, D, H, W, C, ws, ss,
                                         static_cast<cudaStream_t>(stream));
}

int crumpet_unshift_unpartition_crop_norm_3d(void* output, void* normed, int norm_dtype,
                                             const void* windows, const void* residual, int dtype,
                                             const float* weight, const float* bias, float eps,
                                             int64_t B, int64_t D, int64_t H, int64_t W, int64_t C,
                                             int64_t ws_d, int64_t ws_h, int64_t ws_w,
                                             int64_t ss_d, int64_t ss_h, int64_t ss_w,
                                             void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_dtype(norm_dtype)) return e;
  const int64_t ws[3] = {ws_d, ws_h, ws_w}, ss[3] = {ss_d, ss_h, ss_w};
  return launch_unshift_unpartition_crop_norm(output, normed, norm_dtype, windows, residual, dtype,
                                              weight, bias, eps, B, D, H, W, C, ws, ss,
                                              static_cast<cudaStream_t>(stream));
}

int crumpet_patch_merge_norm_3d(void* output, int out_dtype, const void* x, int in_dtype,
                                const float* weight, const float* bias, float eps, int64_t B,
                                int64_t D, int64_t H, int64_t W, int64_t C, const int* parts,
                                void* stream) {
  if (int e = check_dtype(out_dtype)) return e;
  if (int e = check_dtype(in_dtype)) return e;
  return launch_patch_merge_norm(output, out_dtype, x, in_dtype, weight, bias, eps, B, D, H, W, C,
                                 parts, static_cast<cudaStream_t>(stream));
}

int crumpet_window_linear(void* out, const void* x, const void* weight, const float* bias,
                          int dtype, int64_t M, int64_t K, int64_t N, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  return launch_window_linear(out, x, weight, bias, dtype, M, K, N,
                              static_cast<cudaStream_t>(stream));
}

int crumpet_proj_out_norm_3d(void* output, int out_dtype, const void* x, int in_dtype,
                             const float* weight, const float* bias, float eps, int64_t B,
                             int64_t C, int64_t D, int64_t H, int64_t W, void* stream) {
  if (int e = check_dtype(out_dtype)) return e;
  if (int e = check_dtype(in_dtype)) return e;
  return launch_proj_out_norm(output, out_dtype, x, in_dtype, weight, bias, eps, B, C, D, H, W,
                              static_cast<cudaStream_t>(stream));
}

int crumpet_roi_gather(void* out, int out_dtype, const void* volume, int in_dtype, int64_t C,
                       int64_t D, int64_t H, int64_t W, const int64_t* roi_starts, int64_t n,
                       int64_t rd, int64_t rh, int64_t rw, void* stream) {
  if (int e = check_dtype(out_dtype)) return e;
  if (int e = check_dtype(in_dtype)) return e;
  return launch_roi_gather(out, out_dtype, volume, in_dtype, C, D, H, W, roi_starts, n, rd, rh,
                           rw, static_cast<cudaStream_t>(stream));
}

int crumpet_roi_accumulate(float* acc, const void* pred, int pred_dtype, int64_t classes,
                           int64_t D, int64_t H, int64_t W, const int64_t* roi_starts, int64_t n,
                           int64_t rd, int64_t rh, int64_t rw, void* stream) {
  if (int e = check_dtype(pred_dtype)) return e;
  return launch_roi_accumulate(acc, pred, pred_dtype, classes, D, H, W, roi_starts, n, rd, rh, rw,
                               static_cast<cudaStream_t>(stream));
}

int crumpet_roi_argmax(uint8_t* labels, float* logits, const float* acc, const float* count_d,
                       const float* count_h, const float* count_w, int64_t classes, int64_t D,
                       int64_t H, int64_t W, void* stream) {
  return launch_roi_argmax(labels, logits, acc, count_d, count_h, count_w, classes, D, H, W,
                           static_cast<cudaStream_t>(stream));
}

int crumpet_relative_position_bias(void* bias, int out_dtype, const void* table, int table_dtype,
                                   int64_t table_rows, int64_t H, const int* pairs, int64_t npairs,
                                   void* stream) {
  if (int e = check_dtype(out_dtype)) return e;
  if (int e = check_dtype(table_dtype)) return e;
  if (H < 0 || npairs < 0) return set_error(kErrInvalid, "H and npairs must be non-negative");
  if (H == 0 || npairs == 0) return kOk;
  if (table_rows < 1 || table_rows > 0x7fffffff || npairs > 0x7fffffff || H > 0xffff)
    return set_error(kErrInvalid, "relative position bias: table_rows, npairs or H out of range");
  if (!bias || !table || !pairs) return set_error(kErrInvalid, "null tensor pointer");
  return launch_relative_position_bias(bias, out_dtype, table, table_dtype, table_rows, pairs,
                                       npairs, H, static_cast<cudaStream_t>(stream));
}

int crumpet_relative_position_bias_backward(void* grad_table, int table_dtype, int64_t H,
                                            const void* grad, int grad_dtype, const int* order,
                                            int64_t npairs, const int* items, int64_t n_items,
                                            const int* multi, int64_t n_multi, float* partial,
                                            void* stream) {
  return crumpet_relative_position_bias_backward_rows(grad_table, table_dtype, 0x7fffffff, H, grad,
                                                      grad_dtype, order, npairs, items, n_items,
                                                      multi, n_multi, partial, stream);
}

int crumpet_relative_position_bias_backward_rows(void* grad_table, int table_dtype,
                                                 int64_t table_rows, int64_t H, const void* grad,
                                                 int grad_dtype, const int* order, int64_t npairs,
                                                 const int* items, int64_t n_items,
                                                 const int* multi, int64_t n_multi, float* partial,
                                                 void* stream) {
  if (int e = check_dtype(table_dtype)) return e;
  if (int e = check_dtype(grad_dtype)) return e;
  if (H < 0 || npairs < 0 || n_items < 0 || n_multi < 0)
    return set_error(kErrInvalid, "H, npairs, n_items and n_multi must be non-negative");
  if (H == 0 || n_items == 0) return kOk;
  if (table_rows < 0 || table_rows > 0x7fffffff || npairs > 0x7fffffff || H > 0xffff ||
      n_items > 0x7fffffff || n_multi > 0x7fffffff)
    return set_error(kErrInvalid, "relative position bias: npairs, H or items out of range");
  if (!grad_table || !items || (npairs > 0 && (!grad || !order)) ||
      (n_multi > 0 && (!multi || !partial)))
    return set_error(kErrInvalid, "null tensor pointer");
  BiasGradArgs a{};
  a.grad_table = grad_table;
  a.table_dtype = table_dtype;
  a.table_rows = table_rows;
  a.grad = grad;
  a.grad_dtype = grad_dtype;
  a.npairs = npairs;
  a.H = H;
  a.order = order;
  a.items = items;
  a.multi = multi;
  a.n_items = n_items;
  a.n_multi = n_multi;
  a.partial = partial;
  return launch_relative_position_bias_grad(a, static_cast<cudaStream_t>(stream));
}

int64_t crumpet_window_attention_backward_shares(int64_t B, int64_t H, int64_t N, int64_t head_dim,
                                                 int dtype) {
  if (B < 0 || H < 1 || N < 1) return 0;
  return attention_grad_tensor_path(dtype, H, N, head_dim)
             ? attention_grad_shares(B, H, N)
             : attention_grad_shares_simt(B, H, N, head_dim, dtype);
}

}  // extern "C"

namespace {

// Checks of the packed-qkv attention by pairs, forward and backward
int check_train_attention(int dtype, int64_t B, int64_t H, int64_t N, int64_t head_dim, float scale,
                          int64_t table_rows, const int64_t* nw, const int64_t* ws,
                          const int64_t* ss) {
  if (int e = check_dtype(dtype)) return e;
  if (!simt_attention_head_dim(head_dim))
    return set_error(kErrUnsupported,
                     "window attention requires a power-of-two head_dim between 16 and 256");
  if (B < 0 || H < 1 || N < 1) return set_error(kErrInvalid, "B must be >= 0, H and N >= 1");
  if (!(scale > 0.f) || !(scale < 1e30f))
    return set_error(kErrUnsupported, "window attention requires a finite scale > 0");
  if (B > 0x7fffffff || H > 0xffff || N > 46340)
    return set_error(kErrInvalid, "B, H or N too large");
  if (table_rows < 1) return set_error(kErrInvalid, "relative position bias table has no rows");
  if (table_rows > 0x7fffffff) return set_error(kErrInvalid, "relative position bias table too large");
  if ((ss[0] | ss[1] | ss[2]) == 0) return kOk;
  int64_t windows = 1;
  for (int a = 0; a < 3; ++a) {
    if (nw[a] < 1 || ws[a] < 1 || ws[a] > N)
      return set_error(kErrInvalid, "analytic mask geometry does not match N");
    if (nw[a] > 0xffff) return set_error(kErrInvalid, "too many windows per axis");
    if (ss[a] < 0 || ss[a] >= ws[a])
      return set_error(kErrInvalid, "analytic mask shift must satisfy 0 <= shift < window");
    windows *= nw[a];
  }
  if (ws[0] * ws[1] * ws[2] != N)
    return set_error(kErrInvalid, "analytic mask geometry does not match N");
  if (windows > 0x7fffffff) return set_error(kErrInvalid, "too many windows");
  return kOk;
}

AttnGradArgs train_args(const void* qkv, const void* bias_table, int table_f32, int64_t table_rows,
                        const int* pairs, const int64_t* nw, const int64_t* ws, const int64_t* ss, int dtype,
                        int64_t B, int64_t H, int64_t N, int64_t head_dim, float scale) {
  AttnGradArgs a{};
  a.qkv = qkv;
  a.table = bias_table;
  a.table_f32 = table_f32 != 0 || dtype == kF32;
  a.table_rows = table_rows;
  a.pairs = pairs;
  for (int x = 0; x < 3; ++x) {
    a.nwin[x] = nw[x];
    a.win[x] = ws[x];
    a.shift[x] = ss[x];
  }
  a.B = B;
  a.H = H;
  a.N = N;
  a.head_dim = head_dim;
  a.shares = 1;
  a.scale = scale;
  a.dtype = dtype;
  return a;
}

}  // namespace

extern "C" {

int crumpet_swin_window_attention_qkv_pairs(void* out, const void* qkv, const void* bias_table,
                                            int table_f32, int64_t table_rows, const int* pairs,
                                            int64_t nw_d, int64_t nw_h, int64_t nw_w, int64_t ws_d,
                                            int64_t ws_h, int64_t ws_w, int64_t ss_d, int64_t ss_h,
                                            int64_t ss_w, int dtype, int64_t B, int64_t H,
                                            int64_t N, int64_t head_dim, float scale,
                                            void* stream) {
  const int64_t nw[3] = {nw_d, nw_h, nw_w}, ws[3] = {ws_d, ws_h, ws_w}, ss[3] = {ss_d, ss_h, ss_w};
  if (int e = check_train_attention(dtype, B, H, N, head_dim, scale, table_rows, nw, ws, ss))
    return e;
  if (B == 0) return kOk;
  if (!out || !qkv || !bias_table || !pairs) return set_error(kErrInvalid, "null tensor pointer");
  const AttnGradArgs a = train_args(qkv, bias_table, table_f32, table_rows, pairs, nw, ws, ss, dtype,
                                    B, H, N, head_dim, scale);
  return launch_attention_train_simt(a, out, static_cast<cudaStream_t>(stream));
}

int crumpet_swin_window_attention_qkv_backward(
    void* grad_qkv, float* grad_bias, float* stats, const void* grad_out, const void* qkv,
    const void* bias_table, int table_f32, int64_t table_rows, const int* pairs, int64_t shares,
    int64_t nw_d, int64_t nw_h, int64_t nw_w, int64_t ws_d, int64_t ws_h, int64_t ws_w,
    int64_t ss_d, int64_t ss_h, int64_t ss_w, int dtype, int64_t B, int64_t H, int64_t N,
    int64_t head_dim, float scale, void* stream) {
  const int64_t nw[3] = {nw_d, nw_h, nw_w}, ws[3] = {ws_d, ws_h, ws_w}, ss[3] = {ss_d, ss_h, ss_w};
  if (int e = check_train_attention(dtype, B, H, N, head_dim, scale, table_rows, nw, ws, ss))
    return e;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (shares < 1 || shares > 0xffff || shares > (B > 0 ? B : 1))
    return set_error(kErrInvalid, "shares must be between 1 and the number of windows");
  if (H * ((N + 63) / 64) * shares > 0x7fffffff)
    return set_error(kErrInvalid, "too many windows x heads for one launch");
  if (!grad_bias) return set_error(kErrInvalid, "null tensor pointer");
  if (B == 0) {  // no window: no gradient of the bias
    const cudaError_t e = cudaMemsetAsync(grad_bias, 0, size_t(H * N * N) * sizeof(float), on);
    return e == cudaSuccess ? kOk : set_cuda_error(e, "window attention backward memset");
  }
  if (!grad_qkv || !stats || !grad_out || !qkv || !bias_table || !pairs)
    return set_error(kErrInvalid, "null tensor pointer");
  if (reinterpret_cast<uintptr_t>(stats) & 15u)
    return set_error(kErrInvalid, "stats must be 16-byte aligned");
  AttnGradArgs a = train_args(qkv, bias_table, table_f32, table_rows, pairs, nw, ws, ss, dtype, B, H,
                              N, head_dim, scale);
  a.grad_qkv = grad_qkv;
  a.grad_bias = grad_bias;
  a.stats = stats;
  a.grad_out = grad_out;
  a.shares = shares;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(grad_qkv) |
                         reinterpret_cast<uintptr_t>(grad_out) | reinterpret_cast<uintptr_t>(qkv);
  const bool tensor = attention_grad_tensor_path(dtype, H, N, head_dim) && (bits & 15u) == 0 &&
                      scale >= kTensorMinScale;
  if (int e = tensor ? launch_attention_grad(a, on) : launch_attention_grad_simt(a, on)) return e;
  return launch_sum_shares(grad_bias, shares, H * N * N, on);
}

namespace {

int check_norm_gate(int dtype, int stream_dtype, const float* row_scale, int64_t samples,
                    const float* post_w, const float* post_b, float eps, int64_t M, int64_t C) {
  if (int e = check_dtype(dtype)) return e;
  if (stream_dtype != dtype && stream_dtype != kF32)
    return set_error(kErrInvalid, "the residual stream must be float32 or of the branch's dtype");
  if (M < 0 || C < 1 || C > 4096) return set_error(kErrInvalid, "norm_gate_residual needs 1 <= C <= 4096");
  if (!(eps > 0.f)) return set_error(kErrInvalid, "eps must be positive");
  if (row_scale && (samples < 1 || M % samples))
    return set_error(kErrInvalid, "the rows must divide evenly among the samples of row_scale");
  if ((post_w == nullptr) != (post_b == nullptr))
    return set_error(kErrInvalid, "post weight and bias must both be given or both be NULL");
  return kOk;
}

}  // namespace

int crumpet_norm_gate_residual(void* out, void* normed, const void* branch, const void* residual,
                               int dtype, int stream_dtype, const float* gate,
                               const float* row_scale, int64_t samples, const float* post_w,
                               const float* post_b, const float* pre_w, const float* pre_b,
                               float eps, int64_t M, int64_t C, void* stream) {
  if (int e = check_norm_gate(dtype, stream_dtype, row_scale, samples, post_w, post_b, eps, M, C))
    return e;
  if ((pre_w == nullptr) != (pre_b == nullptr))
    return set_error(kErrInvalid, "pre weight and bias must both be given or both be NULL");
  if (M == 0) return kOk;
  if (!out || !branch || !residual || (pre_w && !normed))
    return set_error(kErrInvalid, "null tensor pointer");
  NormGateArgs n{};
  n.branch = branch;
  n.residual = residual;
  n.out = out;
  n.normed = normed;
  n.gate = gate;
  n.row_scale = row_scale;
  n.post_w = post_w;
  n.post_b = post_b;
  n.pre_w = pre_w;
  n.pre_b = pre_b;
  n.M = M;
  n.C = C;
  n.samples = row_scale ? samples : 1;
  n.eps = eps;
  n.dtype = dtype;
  n.stream_dtype = stream_dtype;
  return launch_norm_gate(n, static_cast<cudaStream_t>(stream));
}

int64_t crumpet_norm_gate_residual_backward_partials(int64_t M, int64_t C) {
  return norm_gate_backward_partials(M, C);
}

int crumpet_norm_gate_residual_backward(
    void* grad_residual, void* grad_branch, float* grad_gate, float* grad_post_w,
    float* grad_post_b, float* grad_pre_w, float* grad_pre_b, const void* grad_out,
    const void* grad_normed, const void* out, const void* branch, int dtype, int stream_dtype,
    const float* gate, const float* row_scale, int64_t samples, const float* post_w,
    const float* post_b, const float* pre_w, float eps, float* partial, int64_t M, int64_t C,
    void* stream) {
  if (int e = check_norm_gate(dtype, stream_dtype, row_scale, samples, post_w, post_b, eps, M, C))
    return e;
  if ((gate && !grad_gate) || (post_w && (!grad_post_w || !grad_post_b)) ||
      (pre_w && (!grad_pre_w || !grad_pre_b)))
    return set_error(kErrInvalid, "null tensor pointer");
  if (M == 0) {  // no rows: the sums over them are zero
    float* const sums[5] = {gate ? grad_gate : nullptr, post_w ? grad_post_w : nullptr,
                            post_w ? grad_post_b : nullptr, pre_w ? grad_pre_w : nullptr,
                            pre_w ? grad_pre_b : nullptr};
    for (float* s : sums) {
      if (!s) continue;
      const cudaError_t e =
          cudaMemsetAsync(s, 0, size_t(C) * sizeof(float), static_cast<cudaStream_t>(stream));
      if (e != cudaSuccess) return set_cuda_error(e, "norm gate residual backward memset");
    }
    return kOk;
  }
  if (!grad_residual || !grad_branch || !grad_out || (pre_w && (!grad_normed || !out)) ||
      ((gate || post_w) && !branch) || ((gate || post_w || pre_w) && !partial))
    return set_error(kErrInvalid, "null tensor pointer");
  NormGateArgs n{};
  n.branch = branch;
  n.out = const_cast<void*>(out);  // only read by the backward
  n.grad_out = grad_out;
  n.grad_normed = grad_normed;
  n.grad_residual = grad_residual;
  n.grad_branch = grad_branch;
  n.partial = partial;
  n.grad_gate = grad_gate;
  n.grad_post_w = grad_post_w;
  n.grad_post_b = grad_post_b;
  n.grad_pre_w = grad_pre_w;
  n.grad_pre_b = grad_pre_b;
  n.gate = gate;
  n.row_scale = row_scale;
  n.post_w = post_w;
  n.post_b = post_b;
  n.pre_w = pre_w;
  n.M = M;
  n.C = C;
  n.samples = row_scale ? samples : 1;
  n.eps = eps;
  n.dtype = dtype;
  n.stream_dtype = stream_dtype;
  return launch_norm_gate_backward(n, static_cast<cudaStream_t>(stream));
}

namespace {

int check_kept(int dtype, int64_t M, int64_t C) {
  if (int e = check_dtype(dtype)) return e;
  if (M < 0 || C < 0) return set_error(kErrInvalid, "M and C must be non-negative");
  if (C > (1 << 24)) return set_error(kErrInvalid, "C must be at most 2^24");
  return kOk;
}

}  // namespace

int crumpet_gelu_checkpoint(void* y, int8_t* kept, uint8_t* scales, const void* x, int dtype,
                            int64_t M, int64_t C, void* stream) {
  if (int e = check_kept(dtype, M, C)) return e;
  if (M == 0 || C == 0) return kOk;
  if (!y || !kept || !scales || !x) return set_error(kErrInvalid, "null tensor pointer");
  return launch_gelu_checkpoint(y, kept, scales, x, dtype, M, C,
                                static_cast<cudaStream_t>(stream));
}

int crumpet_gelu_checkpoint_backward(void* grad_x, void* again, const void* grad_y,
                                     const int8_t* kept, const uint8_t* scales, int dtype,
                                     int64_t M, int64_t C, void* stream) {
  if (int e = check_kept(dtype, M, C)) return e;
  if (M == 0 || C == 0) return kOk;
  if (!grad_x || !again || !grad_y || !kept || !scales)
    return set_error(kErrInvalid, "null tensor pointer");
  return launch_gelu_checkpoint_backward(grad_x, again, grad_y, kept, scales, dtype, M, C,
                                         static_cast<cudaStream_t>(stream));
}

int crumpet_restore_activation(void* x, const int8_t* kept, const uint8_t* scales, int dtype,
                               int64_t M, int64_t C, void* stream) {
  if (int e = check_kept(dtype, M, C)) return e;
  if (M == 0 || C == 0) return kOk;
  if (!x || !kept || !scales) return set_error(kErrInvalid, "null tensor pointer");
  return launch_restore_activation(x, kept, scales, dtype, M, C,
                                   static_cast<cudaStream_t>(stream));
}

int crumpet_test_stall_attention(int enable) { return set_attention_test_stall(enable); }

int crumpet_device_status(int clear) {
  const int v = read_device_error(clear != 0);
  if (v < 0) return set_error(kErrCuda, "could not read the device error word");
  return v;
}

}  // extern "C"
