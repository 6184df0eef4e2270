// Launch interfaces of the operators on embedding rows in device memory
// (internal to the library): 8-bit rows and their scores, and the softmax
// loss over a base with its gradient.
#pragma once

#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

namespace px {

enum ElemType { kElemF32 = 0, kElemF16 = 1, kElemBf16 = 2, kElemS8 = 3 };  // 0-2 match PX_F32 ...

// k_gemm.cu
cudaError_t encode_rows_map(CUtensorMap* map, ElemType type, const void* base, int64_t cols, int64_t rows,
                            int64_t pitch, int box_cols, int box_rows, int swizzle);

// ---- 8-bit rows (k_quant.cu) -----------------------------------------------
cudaError_t launch_quantize_rows(const void* x, ElemType type, int64_t n, int d, int64_t ldx, int8_t* codes,
                                 int64_t ldc, float* scales, cudaStream_t stream);
cudaError_t launch_dequantize_rows(const int8_t* codes, int64_t ldc, const float* scales, int64_t n, int d,
                                   ElemType type, void* out, int64_t ldo, cudaStream_t stream);

// ---- 8-bit scores (k_int8.cu) ----------------------------------------------
struct Int8ScoresArgs {
  const int8_t* q;      // m x d codes, row pitch ldq (multiple of 16), 16-byte aligned
  int64_t ldq;
  const float* q_scale; // m
  int64_t m;
  const int8_t* x;      // n x d codes, row pitch ldx (multiple of 16), 16-byte aligned
  int64_t ldx;
  const float* x_scale; // n
  int64_t n;
  int d;
  const float* bias;    // n, or null
  ElemType type;        // of out
  void* out;            // m x n, row stride ldo elements
  int64_t ldo;
};
// Waits for the stream; *out = the error word, which is cleared.
cudaError_t take_int8_error(cudaStream_t stream, unsigned* out);
cudaError_t launch_int8_scores(const Int8ScoresArgs& a, int clusters, cudaStream_t stream);

// ---- softmax loss over a base (k_xent.cu) ----------------------------------
struct XentProblem {
  const void* q;        // t x d, row stride ldq elements (multiple of 8), 16-byte aligned
  int64_t ldq;
  int64_t t;
  const void* rows;     // v x d, row stride ldr
  int64_t ldr;
  int64_t v;
  int d;
  ElemType type;        // kElemF16 or kElemBf16
  const int64_t* targets;
  int64_t ignore_index;
  float scale;
  const float* bias;    // v, or null; 16-byte aligned
};
cudaError_t take_xent_error(cudaStream_t stream, unsigned* out);
int64_t xent_forward_workspace(int64_t t, int64_t v, int clusters);
int64_t xent_backward_workspace(int64_t t, int64_t v, int d, int clusters);
// loss, lse: t each. reduction: 0 none, 1 sum, 2 mean (total the reduced
// loss, divisor what it was divided by; both may be null when reduction is 0).
cudaError_t launch_xent_forward(const XentProblem& p, float* loss, float* lse, int reduction, float* total,
                                float* divisor, void* ws, int clusters, cudaStream_t stream, int* launches);
// grad: the loss's gradient, t values (grad_stride 1) or one (0); divisor: the
// forward's, or null. dq / drows may be null (not wanted).
cudaError_t launch_xent_backward(const XentProblem& p, const float* loss, const float* lse, const float* grad,
                                 int grad_stride, const float* divisor, void* dq, int64_t lddq, void* drows,
                                 int64_t lddr, void* ws, int clusters, cudaStream_t stream, int* launches);

}  // namespace px
