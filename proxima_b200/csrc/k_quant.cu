// 8-bit rows: each embedding row as signed 8-bit codes and one fp32 scale,
//     scale = max_j |x_j| / 127        (fp32 division)
//     code_j = x_j / scale, rounded to nearest, ties to even
// and back (code * scale). The codes are the exactly rounded quotients: a
// product with the reciprocal gives a candidate, and its remainder
// x - code * scale, which one fma computes without rounding, says whether a
// neighbour is nearer. So the codes do not depend on how the division is
// carried out, at the cost of an fma and a compare per value instead of a
// division.
//
// A row of zeros (or one so small that its scale underflows to 0) has scale 0
// and codes 0. A row that holds a NaN or an infinity has scale NaN and codes
// 0, so every score of it is NaN.
//
// Both kernels move bytes and little else, so the layout is chosen for wide
// coalesced accesses: a group of 4 to 32 lanes takes a row, the widest vector
// that the row's address and pitch allow at a time (16 bytes where rows start
// on 16-byte boundaries), the row staying in registers between the maximum
// and the codes, so x is read once. Groups are as small as leaves a lane at
// most four vectors: several short rows share a warp's load instruction.
// 1M x 128 fp32: 104 us to codes and about the same back, 6.2 TB/s, 0.94 of
// what a copy reaches; issue slots are 79% busy, so the exact rounding just
// hides behind the bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "px_rows.cuh"
#include "px_rows.h"

namespace px {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // loads in flight per thread, ahead of the stores

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<1> { using type = uint8_t; };

// The larger of a and |b|; NaN if either is.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// A row's scale, and its values' codes.
struct RowScale {
  float scale, inverse, half, lift;
  __device__ __forceinline__ explicit RowScale(float peak) {
    if (!(peak < __int_as_float(0x7f800000))) {  // NaN or infinity in the row
      scale = __int_as_float(0x7fc00000);
      inverse = half = 0.0f;
      lift = 1.0f;
      return;
    }
    scale = __fdiv_rn(peak, 127.0f);
    // Rows so small that 1 / scale would overflow are taken times 2^96 (a power
    // of two, so nothing is rounded).
    lift = scale < 1e-30f ? 0x1p96f : 1.0f;
    inverse = scale > 0.0f ? __frcp_rn(scale * lift) : 0.0f;
    half = 0.5f * (scale * lift);
  }
  // x / scale rounded to a whole number, as the low byte of the result's bits
  // (1.5 * 2^23 + the number), if `off` comes out below `half`; at or above it
  // the exact quotient may round to a neighbour.
  __device__ __forceinline__ float near(float x, float& off) const {
    const float shifted = fmaf(x, inverse, 12582912.0f);
    // |rest| <= scale * (1/2 + a few ulps): computed without rounding.
    const float rest = fmaf(-(shifted - 12582912.0f), 2.0f * half, x);
    off = fmaxf(off, fabsf(rest));
    return shifted;
  }
  // The code itself, for any value.
  __device__ __forceinline__ int code(float x) const {
    if (inverse == 0.0f) return 0;
    const float xs = x * lift;
    float c = rintf(xs * inverse);
    const float rest = fmaf(-c, 2.0f * half, xs);
    const float far = fabsf(rest);
    if (far > half || (far == half && (__float2int_rn(c) & 1))) c += copysignf(1.0f, rest);
    return __float2int_rn(fminf(fmaxf(c, -127.0f), 127.0f));
  }
};

// The codes of four values, one per byte. The common case takes an fma, an
// addition, an fma and a maximum per value; a value at or past a half, or a
// row that is lifted, goes through code().
__device__ __forceinline__ uint32_t four_codes(const RowScale& r, const float* x) {
  float off = 0.0f;
  const uint32_t a = __float_as_uint(r.near(x[0], off)), b = __float_as_uint(r.near(x[1], off));
  const uint32_t c = __float_as_uint(r.near(x[2], off)), d = __float_as_uint(r.near(x[3], off));
  if (off < r.half && r.lift == 1.0f) return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  uint32_t w = 0;
  for (int j = 0; j < 4; ++j) w |= static_cast<uint32_t>(r.code(x[j]) & 0xff) << (8 * j);
  return w;
}

// VB: bytes per load; NV: loads per lane. A row's values stay in registers, at
// most 32 per lane.
template <typename T, int VB, int NV>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* x, int64_t n, int d, int64_t ldx,
                                                                 int8_t* codes, int64_t ldc, float* scales, int group,
                                                                 bool vec_out) {
  constexpr int VE = VB / static_cast<int>(sizeof(T));
  using W = typename Word<VB>::type;
  wait_for_previous();
  let_next_start();
  const int lane = threadIdx.x & (group - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / group;
  const bool live = row < n;  // a dead group still takes part in the shuffles
  const T* xr = x + (live ? row : 0) * ldx;
  const int nvec = (d + VE - 1) / VE;
  float v[NV][VE];
  float peak = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * group + lane) * VE;
    if (live && at + VE <= d) {
      const W w = *reinterpret_cast<const W*>(xr + at);
      const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
      for (int j = 0; j < VE; ++j) v[i][j] = to_f32(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) v[i][j] = live && at + j < d ? to_f32(xr[at + j]) : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) peak = max_abs(peak, v[i][j]);
  for (int s = group >> 1; s > 0; s >>= 1) peak = max_abs(peak, __shfl_xor_sync(0xffffffffu, peak, s));
  if (!live) return;
  const RowScale r(peak);
  if (lane == 0) scales[row] = r.scale;
  int8_t* out = codes + row * ldc;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vec = i * group + lane;
    if (vec >= nvec) break;
    const int at = vec * VE;
    using C = typename Word<VE>::type;
    if (vec_out && at + VE <= d) {
      if constexpr (VE >= 4) {
        uint32_t w[VE / 4];
#pragma unroll
        for (int j = 0; j < VE / 4; ++j) w[j] = four_codes(r, &v[i][4 * j]);
        *reinterpret_cast<C*>(out + at) = *reinterpret_cast<const C*>(w);
      } else {
        C w;
        int8_t* e = reinterpret_cast<int8_t*>(&w);
#pragma unroll
        for (int j = 0; j < VE; ++j) e[j] = static_cast<int8_t>(r.code(v[i][j]));
        *reinterpret_cast<C*>(out + at) = w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j)
        if (at + j < d) out[at + j] = static_cast<int8_t>(r.code(v[i][j]));
    }
  }
}

// Rows longer than a group's registers hold: a block per row, which reads the
// row twice (the second time from cache).
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_long_rows_kernel(const T* x, int64_t n, int d, int64_t ldx,
                                                                      int8_t* codes, int64_t ldc, float* scales) {
  __shared__ float s_peak[kThreads / 32];
  wait_for_previous();
  let_next_start();
  for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float peak = 0.0f;
#pragma unroll 8
    for (int j = threadIdx.x; j < d; j += kThreads) peak = max_abs(peak, to_f32(xr[j]));
    for (int s = 16; s > 0; s >>= 1) peak = max_abs(peak, __shfl_xor_sync(0xffffffffu, peak, s));
    if ((threadIdx.x & 31) == 0) s_peak[threadIdx.x >> 5] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) peak = max_abs(peak, s_peak[w]);
    __syncthreads();
    const RowScale r(peak);
    if (threadIdx.x == 0) scales[row] = r.scale;
    int8_t* out = codes + row * ldc;
    for (int j0 = threadIdx.x; j0 < d; j0 += kAhead * kThreads) {
      float v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = j0 + i * kThreads < d ? to_f32(xr[j0 + i * kThreads]) : 0.0f;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (j0 + i * kThreads < d) out[j0 + i * kThreads] = static_cast<int8_t>(r.code(v[i]));
    }
  }
}

// Contiguous rows (ldx = d) that begin off 16-byte boundaries, or are longer
// than the registers of a group: a block takes `rows` of them as one span,
// which it reads into shared memory in aligned 16-byte pieces; groups of lanes
// then take a row each from there, value by value, and store its codes in words
// (`words`: they lie on 4-byte boundaries). 199k x 619 fp16 in 204 us, 115k x
// 803 fp32 in 148; value by value from global memory 528 and 256.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_span_kernel(const T* x, int64_t n, int d, int8_t* codes, int64_t ldc,
                                                                 float* scales, int rows, int group, bool words) {
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  extern __shared__ __align__(16) unsigned char s_bytes[];
  T* s_x = reinterpret_cast<T*>(s_bytes);
  wait_for_previous();
  let_next_start();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows, first = row0 * d, all = n * d;
  const int here = static_cast<int>(n - row0 < rows ? n - row0 : rows);
  // Value e of the span lies at s_x[past + e].
  const int past = static_cast<int>(reinterpret_cast<uintptr_t>(x + first) % 16 / sizeof(T));
  const int pieces = (past + here * d + kPiece - 1) / kPiece;
  for (int p0 = threadIdx.x; p0 < pieces; p0 += kAhead * kThreads) {
    uint4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = p0 + i * kThreads;
      const int64_t at = first - past + static_cast<int64_t>(p) * kPiece;
      if (p < pieces && at >= 0 && at + kPiece <= all) w[i] = *reinterpret_cast<const uint4*>(x + at);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = p0 + i * kThreads;
      const int64_t at = first - past + static_cast<int64_t>(p) * kPiece;
      if (p >= pieces) break;
      if (at >= 0 && at + kPiece <= all) {
        *reinterpret_cast<uint4*>(s_x + p * kPiece) = w[i];
      } else {  // the array's ends
        for (int j = 0; j < kPiece; ++j)
          if (at + j >= 0 && at + j < all) s_x[p * kPiece + j] = x[at + j];
      }
    }
  }
  __syncthreads();
  const int pitch = (d + 3) & ~3;
  int8_t* s_codes = reinterpret_cast<int8_t*>(s_bytes + (static_cast<size_t>(rows) * d * sizeof(T) + 31) / 16 * 16);
  const int lane = threadIdx.x & (group - 1), groups = kThreads / group;
  for (int r0 = 0; r0 < here; r0 += groups) {
    const int r = r0 + threadIdx.x / group;
    const bool live = r < here;  // a dead group still takes part in the shuffles
    const T* xr = s_x + past + (live ? r : 0) * d;
    float peak = 0.0f;
#pragma unroll 4
    for (int j = lane; j < d; j += group) peak = max_abs(peak, to_f32(xr[j]));
    for (int m = group >> 1; m > 0; m >>= 1) peak = max_abs(peak, __shfl_xor_sync(0xffffffffu, peak, m));
    const RowScale q(peak);
    int8_t* c = s_codes + (live ? r : 0) * pitch;
    if (live) {
      if (lane == 0) scales[row0 + r] = q.scale;
      float off = 0.0f;
#pragma unroll 4
      for (int j = lane; j < d; j += group) c[j] = static_cast<int8_t>(__float_as_uint(q.near(to_f32(xr[j]), off)) & 0xff);
      if (!(off < q.half && q.lift == 1.0f))
        for (int j = lane; j < d; j += group) c[j] = static_cast<int8_t>(q.code(to_f32(xr[j])));
    }
    __syncwarp();
    if (live) {
      int8_t* out = codes + (row0 + r) * ldc;
      const int whole = words ? d & ~3 : 0;
      for (int j = 4 * lane; j < whole; j += 4 * group)
        *reinterpret_cast<uint32_t*>(out + j) = *reinterpret_cast<const uint32_t*>(c + j);
      for (int j = whole + lane; j < d; j += group) out[j] = c[j];
    }
  }
}

// The other way: codes to contiguous rows (ldo = d) off 16-byte boundaries. A
// block takes `rows` of them as one span of at most 2^15 values, a thread an
// aligned 16-byte piece of it at a time, wherever in a row it begins; `words`:
// codes are read as words (their rows lie on 4-byte boundaries). 60k x 1537 to
// fp32 in 109 us; value by value 139, through shared memory 292.
template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize_span_kernel(const int8_t* codes, int64_t ldc, const float* scales,
                                                                   int64_t n, int d, T* out, int rows, bool words) {
  constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
  wait_for_previous();
  let_next_start();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows;
  const int total = static_cast<int>(n - row0 < rows ? n - row0 : rows) * d;
  T* o = out + row0 * d;
  codes += row0 * ldc;
  scales += row0;
  const int past = static_cast<int>(reinterpret_cast<uintptr_t>(o) % 16 / sizeof(T));
  const float inverse = 1.0f / static_cast<float>(d);
  // The row of value e < 2^15: e + 1/2 is at least 1/2 / d away from where the
  // row changes, far more than the product's error.
  auto row_of = [&](int e) { return static_cast<int>((static_cast<float>(e) + 0.5f) * inverse); };
  for (int p = threadIdx.x; p * kPiece < past + total; p += kThreads) {
    const int at = p * kPiece - past;
    const int row = at > 0 ? row_of(at) : 0, j = at - row * d;
    if (at >= 0 && j + kPiece <= d) {  // within one row
      const int8_t* c = codes + row * ldc + j;
      uint32_t w[kPiece / 4];
      if (words && (j & ~3) + kPiece + 4 <= d) {
        const uint32_t* c4 = reinterpret_cast<const uint32_t*>(c - (j & 3));
        uint32_t lo = c4[0];
#pragma unroll
        for (int i = 0; i < kPiece / 4; ++i) {
          const uint32_t hi = c4[i + 1];
          w[i] = __funnelshift_r(lo, hi, 8 * (j & 3));
          lo = hi;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPiece / 4; ++i) {
          w[i] = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[i] |= static_cast<uint32_t>(static_cast<uint8_t>(c[4 * i + k])) << (8 * k);
        }
      }
      const float s = scales[row];
      uint4 v;
      T* e = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
        e[i] = from_f32<T>(static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)))) * s);
      *reinterpret_cast<uint4*>(o + at) = v;
    } else {  // where a row or the span ends
      __align__(16) T e[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        if (at + i < 0 || at + i >= total) continue;
        const int er = row_of(at + i);
        e[i] = from_f32<T>(static_cast<float>(codes[er * ldc + (at + i - er * d)]) * scales[er]);
      }
      if (at >= 0 && at + kPiece <= total) {
        *reinterpret_cast<uint4*>(o + at) = *reinterpret_cast<const uint4*>(e);
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
          if (at + i >= 0 && at + i < total) o[at + i] = e[i];
      }
    }
  }
}

// VE codes at a time, AHEAD loads before their stores; a group of lanes takes a
// row, as above.
template <typename T, int VE, int AHEAD>
__global__ void __launch_bounds__(kThreads) dequantize_rows_kernel(const int8_t* codes, int64_t ldc, const float* scales,
                                                                   int64_t n, int d, T* out, int64_t ldo, int group) {
  using C = typename Word<VE>::type;
  using W = typename Word<VE * static_cast<int>(sizeof(T))>::type;
  wait_for_previous();
  let_next_start();
  const int lane = threadIdx.x & (group - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / group;
  if (row >= n) return;
  const float s = scales[row];
  const int8_t* c = codes + row * ldc;
  T* o = out + row * ldo;
  const int step = group * VE;
  for (int at0 = lane * VE; at0 < d; at0 += AHEAD * step) {
    C w[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (at0 + i * step + VE <= d) w[i] = *reinterpret_cast<const C*>(c + at0 + i * step);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = at0 + i * step;
      if (at + VE <= d) {
        const int8_t* e = reinterpret_cast<const int8_t*>(&w[i]);
        W r;
        T* p = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < VE; ++j) p[j] = from_f32<T>(static_cast<float>(e[j]) * s);
        *reinterpret_cast<W*>(o + at) = r;
      } else {
        for (int j = at; j < d; ++j) o[j] = from_f32<T>(static_cast<float>(c[j]) * s);
      }
    }
  }
}

// Lanes per row: the fewest (4 to 32) that leave a lane at most `most` vectors.
int group_for(int64_t vectors, int most) {
  int g = 4;
  while (g < 32 && g * most < vectors) g *= 2;
  return g;
}

// Rows of `bytes` that a block takes as one span: about 16 KB of them, a
// multiple of the `at_once` that its groups take, and at most 1024 (with their
// codes less than 48 KB of shared memory); fewer where the blocks would not
// fill the GPU. 0: a row is too long.
int span_rows(int64_t n, int64_t bytes, int at_once) {
  if (bytes > 32000) return 0;
  int64_t rows = 16384 / bytes;
  const int64_t share = (n + 591) / 592, most = 32000 / bytes;
  rows = rows > at_once ? rows / at_once * at_once : at_once < most ? at_once : most;
  if (rows > share) rows = share;
  if (rows > 1024) rows = 1024;
  return rows > 1 ? static_cast<int>(rows) : 1;
}

bool aligned(const void* p, int64_t pitch, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch % bytes == 0;
}

template <typename T, int VB>
cudaError_t quantize_vec(const T* x, int64_t n, int d, int64_t ldx, int8_t* codes, int64_t ldc, float* scales,
                         cudaStream_t stream) {
  constexpr int VE = VB / static_cast<int>(sizeof(T));
  constexpr int kMost = 32 / VE;  // vectors a lane's registers hold
  const int64_t nvec = (d + VE - 1) / VE;
  if (nvec > 32 * kMost) {
    const int64_t grid = n < 65536 ? n : 65536;
    return launch_after(quantize_long_rows_kernel<T>, grid, kThreads, 0, stream, x, n, d, ldx, codes, ldc, scales);
  }
  const int group = group_for(nvec, 4);
  const int64_t blocks = (n * group + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  auto kern = nvec <= 4 * group ? quantize_rows_kernel<T, VB, 4> : quantize_rows_kernel<T, VB, kMost>;
  return launch_after(kern, blocks, kThreads, 0, stream, x, n, d, ldx, codes, ldc, scales, group,
                      aligned(codes, ldc, VE));
}

template <typename T>
cudaError_t quantize_typed(const T* x, int64_t n, int d, int64_t ldx, int8_t* codes, int64_t ldc, float* scales,
                           cudaStream_t stream) {
  const int64_t pitch = ldx * static_cast<int64_t>(sizeof(T));
  const int group = group_for(d, 16);
  const int rows = span_rows(n, d * static_cast<int64_t>(sizeof(T)), kThreads / group);
  // As spans: long rows, and those of which no load takes four values (us, in
  // vectors and as spans: fp32 1M x 33 141 and 102, 100k x 998 227 and 146, 3M x
  // 7 91 and 132; bf16 700k x 100, four values a load, 100 and 140).
  if ((ldx == d || n == 1) && rows > 0 && (d > 1024 || (d >= 16 && !aligned(x, pitch, 4 * sizeof(T))))) {
    const size_t smem = (static_cast<size_t>(rows) * d * sizeof(T) + 31) / 16 * 16 + static_cast<size_t>(rows) * ((d + 3) & ~3);
    const int64_t blocks = (n + rows - 1) / rows;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_after(quantize_span_kernel<T>, blocks, kThreads, smem, stream, x, n, d, codes, ldc, scales, rows,
                        group, aligned(codes, ldc, 4));
  }
  if (aligned(x, pitch, 16)) return quantize_vec<T, 16>(x, n, d, ldx, codes, ldc, scales, stream);
  if (aligned(x, pitch, 8)) return quantize_vec<T, 8>(x, n, d, ldx, codes, ldc, scales, stream);
  if (aligned(x, pitch, 4)) return quantize_vec<T, 4>(x, n, d, ldx, codes, ldc, scales, stream);
  return quantize_vec<T, static_cast<int>(sizeof(T))>(x, n, d, ldx, codes, ldc, scales, stream);
}

template <typename T, int VE>
cudaError_t dequantize_vec(const int8_t* codes, int64_t ldc, const float* scales, int64_t n, int d, T* out, int64_t ldo,
                           cudaStream_t stream) {
  const int group = group_for((d + VE - 1) / VE, 4);
  const int64_t blocks = (n * group + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  auto kern = group * VE >= d ? dequantize_rows_kernel<T, VE, 1> : dequantize_rows_kernel<T, VE, kAhead>;
  return launch_after(kern, blocks, kThreads, 0, stream, codes, ldc, scales, n, d, out, ldo, group);
}

template <typename T>
cudaError_t dequantize_typed(const int8_t* codes, int64_t ldc, const float* scales, int64_t n, int d, T* out,
                             int64_t ldo, cudaStream_t stream) {
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const int64_t pitch = ldo * static_cast<int64_t>(sizeof(T));
  if (aligned(codes, ldc, VE) && aligned(out, pitch, 16))
    return dequantize_vec<T, VE>(codes, ldc, scales, n, d, out, ldo, stream);
  if (aligned(codes, ldc, 2) && aligned(out, pitch, 2 * static_cast<int>(sizeof(T))))
    return dequantize_vec<T, 2>(codes, ldc, scales, n, d, out, ldo, stream);
  // 1M x 33: 72 us, value by value 99.
  const int rows = span_rows(n, d * static_cast<int64_t>(sizeof(T)), 1);
  if ((ldo == d || n == 1) && rows > 0) {
    const int64_t blocks = (n + rows - 1) / rows;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_after(dequantize_span_kernel<T>, blocks, kThreads, 0, stream, codes, ldc, scales, n, d, out, rows,
                        aligned(codes, ldc, 4));
  }
  return dequantize_vec<T, 1>(codes, ldc, scales, n, d, out, ldo, stream);
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, ElemType type, int64_t n, int d, int64_t ldx, int8_t* codes,
                                 int64_t ldc, float* scales, cudaStream_t stream) {
  switch (type) {
    case kElemF32: return quantize_typed(static_cast<const float*>(x), n, d, ldx, codes, ldc, scales, stream);
    case kElemF16: return quantize_typed(static_cast<const __half*>(x), n, d, ldx, codes, ldc, scales, stream);
    case kElemBf16: return quantize_typed(static_cast<const __nv_bfloat16*>(x), n, d, ldx, codes, ldc, scales, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_dequantize_rows(const int8_t* codes, int64_t ldc, const float* scales, int64_t n, int d,
                                   ElemType type, void* out, int64_t ldo, cudaStream_t stream) {
  switch (type) {
    case kElemF32: return dequantize_typed(codes, ldc, scales, n, d, static_cast<float*>(out), ldo, stream);
    case kElemF16: return dequantize_typed(codes, ldc, scales, n, d, static_cast<__half*>(out), ldo, stream);
    case kElemBf16: return dequantize_typed(codes, ldc, scales, n, d, static_cast<__nv_bfloat16*>(out), ldo, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace px
