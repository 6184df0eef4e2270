// C ABI of the operators on embedding rows in device memory (px.h, "Embedding
// rows"): argument checks and launches. Nothing here allocates, keeps state
// between calls or waits for the GPU (px_rows_status_device aside), so every
// call can be captured into a CUDA graph.
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "px_rows.h"
#include "px_runtime.h"

using namespace px;

namespace {

// The 32-bit sums of an 8-bit product hold 2^31 / 128^2 products.
constexpr int32_t kInt8MaxDim = 131071;
constexpr int64_t kMaxRows = 0x7fffff00;  // TMA coordinates are 32-bit

bool is_type(int32_t t) { return t == PX_F32 || t == PX_F16 || t == PX_BF16; }
int64_t size_of(int32_t t) { return t == PX_F32 ? 4 : 2; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

px_status check_device(int32_t device) {
  int count = 0;
  cudaError_t e = cudaGetDeviceCount(&count);
  if (e != cudaSuccess || count == 0) {
    cudaGetLastError();
    return set_error(PX_ECUDA, std::string("no CUDA device available: ") +
                                   (e == cudaSuccess ? "device count is 0" : cudaGetErrorString(e)));
  }
  if (device < 0 || device >= count)
    return set_error(PX_EINVAL, "device ordinal " + std::to_string(device) +
                                    " out of range (visible devices: " + std::to_string(count) + ")");
  return PX_OK;
}

px_status check_rows(int64_t n, int32_t dim, const char* what) {
  if (dim <= 0) return set_error(PX_EINVAL, "dim must be > 0");
  if (n < 0) return set_error(PX_EINVAL, std::string(what) + " must be >= 0");
  if (n > kMaxRows) return set_error(PX_EUNSUPPORTED, std::string(what) + " must be < 2^31 - 256");
  return PX_OK;
}

// An operand that TMA reads: rows on 16-byte boundaries.
px_status check_tiled(const void* p, int64_t ld, int64_t elem, int32_t dim, const char* what) {
  if (p == nullptr) return set_error(PX_EINVAL, "null buffer");
  if (ld < dim) return set_error(PX_EINVAL, std::string(what) + ": the row stride is less than dim");
  if (!aligned16(p) || ld * elem % 16 != 0)
    return set_error(PX_EINVAL, std::string(what) + ": rows must start on 16-byte boundaries");
  // The tensor map's limit on a stride.
  if (ld * elem >= (int64_t(1) << 40)) return set_error(PX_EUNSUPPORTED, std::string(what) + ": the row stride is too large");
  return PX_OK;
}

// Pointers of whole elements.
px_status check_aligned(std::initializer_list<const void*> ps, uintptr_t bytes, const char* what) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
      return set_error(PX_EINVAL, std::string(what) + ": misaligned for its type");
  return PX_OK;
}

// Tiles are numbered in 32 bits.
px_status check_tiles(int64_t a, int64_t b, const char* what) {
  if (((a + 255) / 256) * ((b + 255) / 256) > 0x7fffffff)
    return set_error(PX_EUNSUPPORTED, std::string(what) + " is too large");
  return PX_OK;
}

px_status check_xent(int64_t t, int64_t v, int32_t dim, const void* q, int64_t ldq, const void* rows, int64_t ldr,
                     int32_t type, const int64_t* targets, float scale, const float* bias) {
  px_status s = check_rows(t, dim, "t");
  if (s == PX_OK) s = check_rows(v, dim, "v");
  if (s != PX_OK) return s;
  if (v == 0) return set_error(PX_EINVAL, "a softmax needs at least one base row");
  if (type != PX_F16 && type != PX_BF16)
    return set_error(type == PX_F32 ? PX_EUNSUPPORTED : PX_EINVAL, "queries and rows must be PX_F16 or PX_BF16");
  if (!(scale > 0.0f) || std::isinf(scale)) return set_error(PX_EINVAL, "scale must be positive and finite");
  // Logits are taken in log2 units: scale * log2(e) has to be a number.
  if (scale >= 0x1p127f) return set_error(PX_EINVAL, "scale must be below 2^127");
  if (t == 0) return PX_OK;
  s = check_tiled(q, ldq, 2, dim, "queries");
  if (s == PX_OK) s = check_tiled(rows, ldr, 2, dim, "rows");
  if (s != PX_OK) return s;
  if (targets == nullptr) return set_error(PX_EINVAL, "null buffer");
  s = check_aligned({targets}, 8, "targets");
  if (s == PX_OK) s = check_tiles(t, v, "t * v");
  if (s == PX_OK) s = check_tiles(t > v ? t : v, dim, "dim");
  if (s != PX_OK) return s;
  if (bias != nullptr && !aligned16(bias)) return set_error(PX_EINVAL, "bias must be 16-byte aligned");
  return PX_OK;
}

XentProblem xent_problem(const void* q, int64_t ldq, int64_t t, const void* rows, int64_t ldr, int64_t v, int32_t dim,
                         int32_t type, const int64_t* targets, int64_t ignore_index, float scale, const float* bias) {
  XentProblem p;
  p.q = q;
  p.ldq = ldq;
  p.t = t;
  p.rows = rows;
  p.ldr = ldr;
  p.v = v;
  p.d = dim;
  p.type = static_cast<ElemType>(type);
  p.targets = targets;
  p.ignore_index = ignore_index;
  p.scale = scale;
  p.bias = bias;
  return p;
}

}  // namespace

extern "C" {

PX_API px_status px_quantize_rows_device(int32_t device, const void* x, int32_t type, int64_t n, int32_t dim,
                                         int64_t ldx, int8_t* codes, int64_t ldc, float* scales, void* stream) {
  px_status s = check_rows(n, dim, "n");
  if (s != PX_OK) return s;
  if (!is_type(type)) return set_error(PX_EINVAL, "type must be PX_F32, PX_F16 or PX_BF16");
  if (n == 0) return PX_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return set_error(PX_EINVAL, "null buffer");
  if (ldx < dim || ldc < dim) return set_error(PX_EINVAL, "a row stride is less than dim");
  s = check_aligned({x}, size_of(type), "x");
  if (s == PX_OK) s = check_aligned({scales}, 4, "scales");
  if (s != PX_OK) return s;
  if ((s = check_device(device)) != PX_OK) return s;
  DeviceGuard dg(device);
  cudaError_t e = launch_quantize_rows(x, static_cast<ElemType>(type), n, dim, ldx, codes, ldc, scales,
                                       static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) g_launches += 1;
  return cuda_status(e, "quantize_rows launch");
}

PX_API px_status px_dequantize_rows_device(int32_t device, const int8_t* codes, int64_t ldc, const float* scales,
                                           int64_t n, int32_t dim, int32_t type, void* out, int64_t ldo,
                                           void* stream) {
  px_status s = check_rows(n, dim, "n");
  if (s != PX_OK) return s;
  if (!is_type(type)) return set_error(PX_EINVAL, "type must be PX_F32, PX_F16 or PX_BF16");
  if (n == 0) return PX_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr) return set_error(PX_EINVAL, "null buffer");
  if (ldc < dim || ldo < dim) return set_error(PX_EINVAL, "a row stride is less than dim");
  s = check_aligned({out}, size_of(type), "out");
  if (s == PX_OK) s = check_aligned({scales}, 4, "scales");
  if (s != PX_OK) return s;
  if ((s = check_device(device)) != PX_OK) return s;
  DeviceGuard dg(device);
  cudaError_t e = launch_dequantize_rows(codes, ldc, scales, n, dim, static_cast<ElemType>(type), out, ldo,
                                         static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) g_launches += 1;
  return cuda_status(e, "dequantize_rows launch");
}

PX_API px_status px_int8_scores_device(int32_t device, const int8_t* q, int64_t ldq, const float* q_scales, int64_t m,
                                       const int8_t* x, int64_t ldx, const float* x_scales, int64_t n, int32_t dim,
                                       const float* bias, int32_t type, void* out, int64_t ldo, void* stream) {
  px_status s = check_rows(m, dim, "m");
  if (s == PX_OK) s = check_rows(n, dim, "n");
  if (s != PX_OK) return s;
  if (!is_type(type)) return set_error(PX_EINVAL, "type must be PX_F32, PX_F16 or PX_BF16");
  if (dim > kInt8MaxDim)
    return set_error(PX_EUNSUPPORTED, "dim=" + std::to_string(dim) + " exceeds " + std::to_string(kInt8MaxDim) +
                                          ": a sum of 8-bit products could pass 32 bits");
  if (m == 0 || n == 0) return PX_OK;
  s = check_tiled(q, ldq, 1, dim, "queries");
  if (s == PX_OK) s = check_tiled(x, ldx, 1, dim, "rows");
  if (s != PX_OK) return s;
  if (q_scales == nullptr || x_scales == nullptr || out == nullptr) return set_error(PX_EINVAL, "null buffer");
  if (ldo < n) return set_error(PX_EINVAL, "out: the row stride is less than n");
  s = check_aligned({out}, size_of(type), "out");
  if (s == PX_OK) s = check_aligned({q_scales, x_scales, bias}, 4, "scales or bias");
  if (s == PX_OK) s = check_tiles(m, n, "m * n");
  if (s != PX_OK) return s;
  if ((s = check_device(device)) != PX_OK) return s;
  DeviceGuard dg(device);
  Int8ScoresArgs a;
  a.q = q;
  a.ldq = ldq;
  a.q_scale = q_scales;
  a.m = m;
  a.x = x;
  a.ldx = ldx;
  a.x_scale = x_scales;
  a.n = n;
  a.d = dim;
  a.bias = bias;
  a.type = static_cast<ElemType>(type);
  a.out = out;
  a.ldo = ldo;
  cudaError_t e = launch_int8_scores(a, gemm_pair_clusters(device), static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) g_launches += 1;
  return cuda_status(e, "int8_scores launch");
}

PX_API int64_t px_softmax_xent_workspace_bytes(int32_t device, int64_t t, int64_t v, int32_t dim, int32_t backward) {
  if (t < 0 || v < 0 || dim <= 0 || t > kMaxRows || v > kMaxRows) return 0;
  if (check_tiles(t, v, "t * v") != PX_OK || check_tiles(t > v ? t : v, dim, "dim") != PX_OK) return 0;
  if (t == 0 || v == 0) return 0;
  DeviceGuard dg(device);
  const int clusters = gemm_pair_clusters(device);
  return backward ? xent_backward_workspace(t, v, dim, clusters) : xent_forward_workspace(t, v, clusters);
}

PX_API px_status px_softmax_xent_device(int32_t device, const void* queries, int64_t ldq, int64_t t, const void* rows,
                                        int64_t ldr, int64_t v, int32_t dim, int32_t type, const int64_t* targets,
                                        int64_t ignore_index, float scale, const float* bias, int32_t reduction,
                                        float* loss, float* lse, float* total, float* divisor, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  px_status s = check_xent(t, v, dim, queries, ldq, rows, ldr, type, targets, scale, bias);
  if (s != PX_OK) return s;
  if (reduction != PX_REDUCE_NONE && reduction != PX_REDUCE_SUM && reduction != PX_REDUCE_MEAN)
    return set_error(PX_EINVAL, "reduction must be PX_REDUCE_NONE, PX_REDUCE_SUM or PX_REDUCE_MEAN");
  if (t == 0) return PX_OK;
  if (loss == nullptr || lse == nullptr || (reduction != PX_REDUCE_NONE && (total == nullptr || divisor == nullptr)))
    return set_error(PX_EINVAL, "null buffer");
  s = check_aligned({loss, lse, total, divisor}, 4, "an output");
  if (s != PX_OK) return s;
  if ((s = check_device(device)) != PX_OK) return s;
  DeviceGuard dg(device);
  const int clusters = gemm_pair_clusters(device);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < xent_forward_workspace(t, v, clusters))
    return set_error(PX_EINVAL, "workspace: 16-byte aligned and px_softmax_xent_workspace_bytes long");
  int launches = 0;
  cudaError_t e = launch_xent_forward(xent_problem(queries, ldq, t, rows, ldr, v, dim, type, targets, ignore_index, scale, bias),
                                      loss, lse, reduction, total, divisor, workspace, clusters,
                                      static_cast<cudaStream_t>(stream), &launches);
  g_launches += launches;
  return cuda_status(e, "softmax_xent launch");
}

PX_API px_status px_softmax_xent_backward_device(int32_t device, const void* queries, int64_t ldq, int64_t t,
                                                 const void* rows, int64_t ldr, int64_t v, int32_t dim, int32_t type,
                                                 const int64_t* targets, int64_t ignore_index, float scale,
                                                 const float* bias, const float* loss, const float* lse,
                                                 const float* grad, int32_t grad_stride, const float* divisor,
                                                 void* grad_queries, int64_t ldgq, void* grad_rows, int64_t ldgr,
                                                 void* workspace, int64_t workspace_bytes, void* stream) {
  px_status s = check_xent(t, v, dim, queries, ldq, rows, ldr, type, targets, scale, bias);
  if (s != PX_OK) return s;
  if (grad_stride != 0 && grad_stride != 1) return set_error(PX_EINVAL, "grad_stride must be 0 or 1");
  if (t == 0 || (grad_queries == nullptr && grad_rows == nullptr)) return PX_OK;
  if (loss == nullptr || lse == nullptr || grad == nullptr) return set_error(PX_EINVAL, "null buffer");
  if ((grad_queries != nullptr && ldgq < dim) || (grad_rows != nullptr && ldgr < dim))
    return set_error(PX_EINVAL, "a row stride is less than dim");
  s = check_aligned({grad_queries, grad_rows}, 2, "a gradient");
  if (s == PX_OK) s = check_aligned({loss, lse, grad, divisor}, 4, "an input");
  if (s != PX_OK) return s;
  if ((s = check_device(device)) != PX_OK) return s;
  DeviceGuard dg(device);
  const int clusters = gemm_pair_clusters(device);
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < xent_backward_workspace(t, v, dim, clusters))
    return set_error(PX_EINVAL, "workspace: 16-byte aligned and px_softmax_xent_workspace_bytes long");
  int launches = 0;
  cudaError_t e = launch_xent_backward(
      xent_problem(queries, ldq, t, rows, ldr, v, dim, type, targets, ignore_index, scale, bias), loss, lse, grad,
      grad_stride, divisor, grad_queries, ldgq, grad_rows, ldgr, workspace, clusters,
      static_cast<cudaStream_t>(stream), &launches);
  g_launches += launches;
  return cuda_status(e, "softmax_xent backward launch");
}

PX_API px_status px_rows_status_device(int32_t device, void* stream) {
  px_status s = check_device(device);
  if (s != PX_OK) return s;
  DeviceGuard dg(device);
  unsigned a = 0, b = 0;
  cudaError_t e = take_int8_error(static_cast<cudaStream_t>(stream), &a);
  if (e == cudaSuccess) e = take_xent_error(static_cast<cudaStream_t>(stream), &b);
  if (e != cudaSuccess) return cuda_status(e, "rows status");
  if (a | b) return set_error(PX_ETIMEOUT, "a device-side wait of a row operator timed out; its results are NaN");
  return PX_OK;
}

}  // extern "C"
