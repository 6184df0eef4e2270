// Softmax cross entropy of queries over a whole base, and its gradient,
// without the t x v matrix of logits:
//     z_ij = scale * q_i . r_j + bias_j
//     loss_i = log sum_j exp z_ij - z_i,y(i)
//     G_ij = g_i (exp(z_ij - lse_i) - [j = y(i)]),  dq = scale * G r,  dr = scale * G^T q
//
// Forward: one pass over the products, whose epilogue keeps a running sum of
// exponentials per query, with its scale, over the other rows; a second kernel
// joins them. The target's own logit stays out of the sum, so the loss is
//     softplus(log sum_{j != y} exp z_ij - z_iy),
// which does not cancel when the target holds nearly all of the softmax. z_iy
// is a dot product of its own in the joining kernel, in fp32 with rounding:
// the tensor cores cut the bits their accumulators cannot hold, an error of
// one sign that a loss near zero would show.
//
// Backward: the base is taken in pieces of columns. For each piece the
// products are computed again, their epilogue writes the piece of G, and two
// more products read it: dq accumulates over the pieces in fp32 slabs (one per
// split of the piece, added to in the same order every time, so results do not
// change from run to run), dr is complete per piece.
// G is kept as the sum of two numbers of the operands' 16-bit type, an entry
// rounded and what the rounding took, and each gradient is the sum of both
// parts' products. One part alone is off by up to 2^-8 of an entry (bf16). The
// entries of a query add up to zero, so where rows with large entries lie near
// one another (a target and its hard negatives), the products cancel and the
// rounding's errors do not: a negative that holds most of the rest, 0.03 of the
// rows' length away from the target, left dq off by 3%. Both parts together are
// within 2^-16 (bf16) or 2^-22 (fp16) of an entry.
// The second part counts where entries are large, and a query has few of those:
// it is kept for blocks of 32 queries x 64 rows with an entry above kLarge of
// its query's gradient, and the products take it for slices with such a block.
// Elsewhere an entry's error is at most 2^-17 of its query's gradient (bf16),
// and the errors of many such entries average out (those of rows that are
// alike to the last bit do not, and come to 2^-8 of what such rows hold).
// Entries are relative to the largest |g_i|, times 2^14 for fp16, whose smallest
// normal would otherwise lie above the probabilities of a large base; an fp16
// entry is held to 2^-39 of the largest |g_i| at best.
// G lies in blocks of 64 columns, each block's rows of 128 bytes behind one
// another, those of the second part after those of the first: what a tile
// writes, and what a load of it reads, is then a run of 16 to 32 KB instead of
// lines a row of G apart. Its rows are padded with zeros to whole K slices of
// dr, its last block's columns likewise.
//
// All three products are one kernel, instantiated per role: CTA pairs
// (tcgen05.mma cta_group::2, kind::f16), 256 M rows per pair, K slices of 64.
// Operands stream through a ring of 16 KB slots (14 in shared memory for the
// forward, 12 for the others, which stage stores beside them), each with its own
// barriers. The MMA warp stays converged and one elected lane issues, so that
// descriptors live in uniform registers: with a lone lane walking the loop the
// tensor pipe waited for its issuer. The three read their operands as they lie: G^T, the base as dq's
// right operand and the queries as dr's are MN-major tiles, so nothing is
// transposed in memory.
//   Logits (kStats, kWeights): 256 x 256 tiles, two accumulators so that the
//   epilogue overlaps the next tile. A pair walks along the base with its
//   queries' slices kept in shared memory (the first seven; d <= 448 keeps
//   all), which halves what it fetches from L2: streaming both operands asks
//   L2 for 64 bytes per SM and clock at the full rate, more than it gives.
//   Tiles are numbered query tile major and dealt to the pairs in equal runs.
//   Gradients (kGradQ, kGradRows): tiles as wide as d up to 512 columns, for
//   the same reason (53 bytes per SM and clock at 384); up to 256 columns the
//   accumulator is doubled.
// 16 epilogue warps: four per TMEM quarter, on 64 columns each (logits) or on
// alternate 32-column blocks (gradients).
//
// Bound: the tensor pipe for d >= 256 or so (2 t v d operations forward, three
// times that backward, of which the logits again are the price of not keeping
// them); the forward at small d by the exponentials (one per logit, 16 per SM
// and clock: 2048 clocks per tile against 512 per slice of products). Computing
// a quarter or three eighths of them by a polynomial on the FMA pipe was slower
// (1000 x 1M x 128: 374 and 396 us against 351 then), though issue slots are 52% busy.
// Measured, bf16: forward 1000 x 1M x 128 327-345 us (2900 clocks per tile), 4096 x
// 100k x 384 1.53 PFLOP/s and, with the epilogue left out, 1.60; past the kept
// slices the operands' way from L2 counts (d = 768: 1.25, 1.30). A training
// step of 1000 x 100k x 384: 355-395 us in two pieces; 8192 x 8192 x 768 (fp16):
// 403-414 us with each query's own row as its target, 489-509 with targets at
// random, so that four slices of G in five have a second part. One part
// throughout: 343 and 418; two throughout: 499 and 551.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "px_rows.cuh"
#include "px_rows.h"

namespace px {

namespace {

// Set when a bounded wait gave up (px_rows_status_device reads and clears it).
__device__ unsigned g_xent_err;

constexpr int kHalf = 128;   // M rows per CTA (TMEM lanes)
constexpr int kTile = 256;   // M rows per pair; N columns of a logits tile
constexpr int kSlice = 64;   // K values per slice: 128 bytes
constexpr int kSlots = 12;       // 16 KB each; the forward stages no stores and has
constexpr int kStatsSlots = 14;  // their 32 KB for slots too
constexpr int kSlot = kHalf * 128;  // 16 KB
constexpr int kKeep = 7;     // query slices kept in shared memory at most
constexpr int kGroups = 4;   // epilogue warps per TMEM quarter
constexpr int kEpiWarps = 4 * kGroups;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kOutBuf = 2048;  // staging of an epilogue warp's stores: 32 rows of 64 bytes
constexpr int kBars = 2 * kStatsSlots + 2 + 2 + 2 + 1;
constexpr size_t kSmem = 1024 + kSlots * kSlot + kEpiWarps * kOutBuf + kBars * 8 + 16;
// An entry of G above this share of its query's gradient is kept in two parts.
constexpr float kLarge = 0x1p-9f;
// A running sum is kept relative to 2^base, base the largest logit of the
// first block; a block whose sum passes kRaise (or is NaN) raises it. Between,
// no maximum is needed: fp32 holds sums of 2^60 as exactly as sums of 1.
constexpr float kRaise = 0x1p60f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

enum Role { kStats, kWeights, kGradQ, kGradRows };

template <int ROLE> struct Shape {
  static constexpr bool LOGITS = ROLE == kStats || ROLE == kWeights;
  static constexpr bool A_MN = ROLE == kGradRows;
  static constexpr bool B_MN = !LOGITS;
  static constexpr int SLOTS = ROLE == kStats ? kStatsSlots : kSlots;
};

// What the backward derives a query's G from.
struct RowGrad {
  const float* loss;
  const float* lse;
  const float* grad;
  const float* top;      // the largest finite |grad| (grad itself when grad_stride is 0)
  const float* divisor;  // or null
  int grad_stride;
  float lift;
};

static_assert(kStatsSlots * kSlot == kSlots * kSlot + kEpiWarps * kOutBuf, "one shared-memory layout");

struct Args {
  int64_t t, v;
  int d;
  int g_rows;            // rows of a part of a block of G
  int g_all;             // rows of the whole array: a load from there on reads zeros
  int m_tiles, n_tiles;
  int tiles;             // logits: m_tiles * n_tiles; gradients: items
  int per_split;         // kGradQ: K slices per split
  int next_m, next_n, next_split;  // gradients: from a pair's tile to its next
  int n_cols;            // N of a tile: 256 (logits), else a multiple of 32 up to 512
  int k_slices;
  int keep;              // logits: query slices kept in shared memory
  int per_slot;          // logits: K slices of the base per ring slot, 1 or 2
  int v0;                // first base row of the piece
  int piece;             // its columns
  int lists;             // kStats: (base, sum) pairs per query
  uint32_t idesc, idesc2;  // of the first 256 columns, and of the rest
  float c;               // scale * log2(e)
  float scale;
  const float* bias;
  const int64_t* targets;
  int64_t ignore_index;
  float2* part;          // kStats: [t][lists] (base, sum): sum * 2^base
  unsigned* counter;     // kStats: cleared for the joining kernel
  RowGrad row;           // kWeights, kGradRows, kGradQ where it is direct
  // Which blocks of G have a second part, a byte each, in eights as the products
  // take them: for dq of [row block][query tile], for dr of [row tile][64 queries].
  uint8_t *parts_q, *parts_r;
  int accumulate;        // kGradQ: to what its slabs hold
  int direct;            // kGradQ: one piece in one split, so the product is the gradient
  uint16_t* out;         // the gradient, where TMA cannot store it
  int64_t ldo;
  int out_row0;          // its row of the product's first
  int tma_out;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// x rounded to the operands' type.
template <bool BF>
__device__ __forceinline__ float rounded(float x) {
  return BF ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
}

__device__ __forceinline__ bool counts(int64_t y, int64_t ignore_index, int64_t v) {
  return y != ignore_index && y >= 0 && y < v;
}

// What gradients are taken relative to. Where all are zero, infinite or NaN,
// they are taken as they are.
__device__ __forceinline__ float top_of(const RowGrad& r) {
  const float top = fabsf(*r.top);
  return top > 0.0f && top < kInf ? top : 1.0f;
}

// A query's factor: its gradient relative to the largest, lifted; 0 for one
// that adds nothing. An infinity or a NaN stays the query's own.
__device__ __forceinline__ float row_factor(const RowGrad& r, bool used, int64_t t) {
  return used ? r.grad[t * r.grad_stride] / top_of(r) * r.lift : 0.0f;
}

// What the products of G are multiplied by at the end.
__device__ __forceinline__ float out_scale(const RowGrad& r, float scale) {
  const float divisor = r.divisor != nullptr ? *r.divisor : 1.0f;
  // A mean over no query: nothing has a part in it, and G is zero.
  if (divisor == 0.0f) return 0.0f;
  return top_of(r) * scale / r.lift / divisor;
}

// The target's entry: exp(-loss) - 1 is its share minus one, without
// cancellation.
__device__ __forceinline__ float target_entry(const RowGrad& r, int64_t t, float factor) {
  return expm1f(-r.loss[t]) * factor;
}

__device__ __forceinline__ float largest(const uint32_t (&v)[32]) {
  float a[10];
#pragma unroll
  for (int i = 0; i < 10; ++i)
    a[i] = max3(__uint_as_float(v[3 * i]), __uint_as_float(v[3 * i + 1]), __uint_as_float(v[3 * i + 2]));
  const float b0 = max3(a[0], a[1], a[2]);
  const float b1 = max3(a[3], a[4], a[5]);
  const float b2 = max3(a[6], a[7], a[8]);
  const float b3 = max3(a[9], __uint_as_float(v[30]), __uint_as_float(v[31]));
  return max2(max3(b0, b1, b2), b3);
}

// The sum of 2^(c * v - base) over a block.
__device__ __forceinline__ float block_sum(const uint32_t (&v)[32], float c, float base) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j & 3] += ex2(fmaf(__uint_as_float(v[j]), c, -base));
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Logit `at`, or those from `from` on, leave a block.
__device__ __forceinline__ void leave_out(uint32_t (&v)[32], int at) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j == at) v[j] = __float_as_uint(-kInf);
}
__device__ __forceinline__ void leave_out_from(uint32_t (&v)[32], int from) {
#pragma unroll
  for (int j = 0; j < 32; ++j)
    if (j >= from) v[j] = __float_as_uint(-kInf);
}

// A row's bias in log2 units. Below about -1.4e31 (a type's lowest value, say) it
// is -inf: the row is left out, as with -inf itself.
__device__ __forceinline__ float bias2(float b) { return b * (kLog2e * 0x1p24f) * 0x1p-24f; }

// Adds the bias: v becomes c * v + bias * log2(e), log2 units. Columns past
// the base count as left out.
__device__ __forceinline__ void add_bias(uint32_t (&v)[32], const float* bias, int left, float c) {
  if (left >= 32) {
    const float4* b4 = reinterpret_cast<const float4*>(bias);
    const F2 up = f2(kLog2e * 0x1p24f, kLog2e * 0x1p24f), down = f2(0x1p-24f, 0x1p-24f), c2 = f2(c, c);
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 b = b4[j / 4];
      float x[4];
      // bias2, two at a time.
      unpack(fma2(f2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), c2, mul2(mul2(f2(b.x, b.y), up), down)), x[0], x[1]);
      unpack(fma2(f2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), c2, mul2(mul2(f2(b.z, b.w), up), down)), x[2], x[3]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[j + k] = __float_as_uint(x[k]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      v[j] = __float_as_uint(j < left ? fmaf(__uint_as_float(v[j]), c, bias2(bias[j])) : -kInf);
  }
}

// A warp's 32 rows x 64 bytes into its staging buffer, as 64-byte swizzle
// lays them out (16-byte piece p of row r at p ^ (r / 2 % 4): eight
// consecutive lanes cover all banks), then one store by lane 0. The caller's
// previous store has been read when this returns from its first wait.
__device__ __forceinline__ void stage_row(uint32_t buf, int lane, const uint32_t (&w)[16]) {
  if (lane == 0) store_wait_read();
  __syncwarp();
  const uint32_t row = buf + lane * 64;
#pragma unroll
  for (int p = 0; p < 4; ++p)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((p ^ ((lane >> 1) & 3)) << 4)), "r"(w[4 * p]),
                 "r"(w[4 * p + 1]), "r"(w[4 * p + 2]), "r"(w[4 * p + 3])
                 : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// Half a warp's 16 rows x 128 bytes likewise, as 128-byte swizzle lays them
// out (piece p of row r at p ^ (r % 8)).
__device__ __forceinline__ void stage_line(uint32_t buf, int lane, int half, const uint32_t (&w)[32]) {
  if (lane == 0) store_wait_read();
  __syncwarp();
  if ((lane >> 4) == half) {
    const int r = lane & 15;
    const uint32_t row = buf + r * 128;
#pragma unroll
    for (int p = 0; p < 8; ++p)
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((p ^ (r & 7)) << 4)), "r"(w[4 * p]),
                   "r"(w[4 * p + 1]), "r"(w[4 * p + 2]), "r"(w[4 * p + 3])
                   : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// A block of stage_row's by plain stores, for an array that TMA cannot address (rows
// that begin or end off 16-byte boundaries): half a warp per row where its pairs of values lie on
// 4-byte boundaries, else a warp per row.
__device__ __forceinline__ void store_staged(uint32_t buf, int lane, uint16_t* out, int64_t ldo, int rows, int cols) {
  const bool words = (reinterpret_cast<uintptr_t>(out) & 3) == 0 && (ldo & 1) == 0;
  constexpr int kAhead = 8;  // reads ahead of the stores
  if (words) {
    const int c = (lane & 15) * 2, half = lane >> 4;
    uint16_t* to = out + half * ldo + c;
#pragma unroll 1
    for (int r0 = half; r0 < 32; r0 += 2 * kAhead) {
      uint32_t x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = r0 + 2 * i;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x[i]) : "r"(buf + r * 64 + (((c >> 3) ^ ((r >> 1) & 3)) << 4) + (c & 7) * 2));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i, to += 2 * ldo) {
        if (r0 + 2 * i >= rows) continue;
        if (c + 1 < cols)
          *reinterpret_cast<uint32_t*>(to) = x[i];
        else if (c < cols)
          *to = static_cast<uint16_t>(x[i]);
      }
    }
  } else {
    uint16_t* to = out + lane;
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += kAhead) {
      uint16_t x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = r0 + i;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x[i]) : "r"(buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i, to += ldo)
        if (r0 + i < rows && lane < cols) *to = x[i];
    }
  }
}

// Where a tile lies. Tiles are numbered along the base, then along the queries
// (logits), or along M, then N, then the splits (gradients). A pair divides its
// first tile's number once and counts on from there; dividing per tile, in the
// epilogue's warps, costs more than it looks (1000 x 1M x 128 forward: 352
// against 327 us), as a division takes the unit that the exponentials keep busy.
struct Place {
  int m, n, split;
};

template <int ROLE>
__device__ __forceinline__ Place place_of(const Args& p, int i) {
  Place at;
  if (Shape<ROLE>::LOGITS) {
    at.m = i / p.n_tiles;
    at.n = i - at.m * p.n_tiles;
    at.split = 0;
  } else {
    const int rest = i / p.m_tiles;
    at.m = i - rest * p.m_tiles;
    at.split = rest / p.n_tiles;
    at.n = rest - at.split * p.n_tiles;
  }
  return at;
}

// To the pair's next tile: the next one, or (gradients) the one `pairs` further,
// which is (next_m, next_n, next_split) on.
template <int ROLE>
__device__ __forceinline__ void advance(const Args& p, Place& at) {
  if (Shape<ROLE>::LOGITS) {
    if (++at.n == p.n_tiles) {
      at.n = 0;
      ++at.m;
    }
  } else {
    at.m += p.next_m;
    at.n += p.next_n;
    at.split += p.next_split;
    if (at.m >= p.m_tiles) {
      at.m -= p.m_tiles;
      ++at.n;
    }
    if (at.n >= p.n_tiles) {
      at.n -= p.n_tiles;
      ++at.split;
    }
  }
}

// A gradient tile's K slices.
template <int ROLE>
__device__ __forceinline__ int first_slice(const Args& p, const Place& at) {
  return ROLE == kGradQ ? at.split * p.per_split : 0;
}
template <int ROLE>
__device__ __forceinline__ int last_slice(const Args& p, const Place& at) {
  return ROLE == kGradQ ? min(p.k_slices, (at.split + 1) * p.per_split) : p.k_slices;
}

// Which blocks of the pair's slice of G have a second part: its eight bytes.
template <int ROLE>
__device__ __forceinline__ uint64_t parts_of(const Args& p, const Place& at, int k) {
  const uint8_t* bytes = ROLE == kGradQ ? p.parts_q + 8 * (static_cast<int64_t>(k) * p.m_tiles + at.m)
                                        : p.parts_r + 8 * (static_cast<int64_t>(at.m) * p.k_slices + k);
  return *reinterpret_cast<const uint64_t*>(bytes);
}

// Logits tiles [first, last) of pair `i` of `n`, and the pair that has tile x.
__host__ __device__ __forceinline__ int run_begin(int64_t tiles, int i, int n) {
  return static_cast<int>(tiles * i / n);
}
__host__ __device__ __forceinline__ int run_of(int64_t tiles, int64_t x, int n) {
  return static_cast<int>(((x + 1) * n - 1) / tiles);
}

template <int ROLE, bool BF, bool BIAS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_part, const Args p) {
  using S = Shape<ROLE>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSlots * kSlot + kEpiWarps * kOutBuf);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(tc::cluster_ctarank());
  const bool leader = rank == 0;
  const uint32_t smem_base = tc::smem_addr(smem);
  auto full_bar = [&](int s) { return tc::smem_addr(&bars[s]); };
  auto empty_bar = [&](int s) { return tc::smem_addr(&bars[kStatsSlots + s]); };
  auto tfull_bar = [&](int a) { return tc::smem_addr(&bars[2 * kStatsSlots + a]); };
  auto tempty_bar = [&](int a) { return tc::smem_addr(&bars[2 * kStatsSlots + 2 + a]); };
  const uint32_t kfull_bar = tc::smem_addr(&bars[2 * kStatsSlots + 4]);   // kept query slices loaded
  const uint32_t kempty_bar = tc::smem_addr(&bars[2 * kStatsSlots + 5]);  // and no longer read
  const uint32_t done_bar = tc::smem_addr(&bars[2 * kStatsSlots + 6]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::SLOTS; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(tfull_bar(a), 1);
      tc::mbar_init(tempty_bar(a), 2 * kEpiWarps);
    }
    tc::mbar_init(kfull_bar, 1);
    tc::mbar_init(kempty_bar, 1);
    tc::mbar_init(done_bar, 1);
    *s_abort = 0;
    tc::fence_mbarrier_init_cluster();
  }
  if (warp == 0 && lane == 0) {
    tc::prefetch_tmap(&tm_a);
    tc::prefetch_tmap(&tm_b);
    if (ROLE != kStats) tc::prefetch_tmap(&tm_out);
    if (S::B_MN) tc::prefetch_tmap(&tm_part);
  }
  if (warp == 1) {
    tc::tmem_alloc_pair(tc::smem_addr(s_tmem), 512);
    tc::tmem_relinquish_pair();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem_base = *s_tmem;
  wait_for_previous();
  let_next_start();
  if (ROLE == kStats && blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0;
  const int cluster = static_cast<int>(tc::cluster_id_x());
  const int nclusters = static_cast<int>(tc::nclusters_x());
  // This pair's tiles: a run (logits), or every nclusters-th item (gradients).
  const int first = S::LOGITS ? run_begin(p.tiles, cluster, nclusters) : cluster;
  const int last = S::LOGITS ? run_begin(p.tiles, cluster + 1, nclusters) : p.tiles;
  const int step = S::LOGITS ? 1 : nclusters;
  // The first `keep` slots of shared memory hold kept query slices, the rest
  // are the ring.
  const int keep = S::LOGITS ? p.keep : 0;
  const int per = S::LOGITS ? p.per_slot : 1;  // slices per ring slot
  const int slot_bytes = per * kSlot;
  const int ring = (S::SLOTS - keep) / per;
  const uint32_t ring_base = smem_base + keep * kSlot;
  // An MN-major B tile: the columns of the first MMA (up to 256) and of the
  // second, in boxes of 64 per CTA.
  const int n_first = min(p.n_cols, kTile);
  const int n_second = p.n_cols - n_first;
  const int accs = p.n_cols > kTile ? 1 : 2;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int64_t loads = 0;
      int slot = 0;
      uint32_t phase = 0;
      int kept = -1;          // query tile whose slices are kept
      Place at = place_of<ROLE>(p, first);
      uint32_t keeps = 0;
      bool ok = true;
      // The next ring slot, armed for both CTAs' bytes; 0 when a wait gave up.
      auto next_slot = [&](uint32_t bytes, uint32_t& fb) -> uint32_t {
        if (!tc::mbar_wait(empty_bar(slot), phase ^ 1, s_abort)) return 0;
        const uint32_t dst = ring_base + slot * slot_bytes;
        fb = tc::mapa_shared(full_bar(slot), 0);
        if (leader) tc::mbar_arrive_expect_tx(full_bar(slot), 2 * bytes);
        ++loads;
        if (++slot == ring) {
          slot = 0;
          phase ^= 1;
        }
        return dst;
      };
      for (int i = first; ok && i < last; i += step) {
        uint32_t fb, dst;
        const int m = at.m, n = at.n;
        if (S::LOGITS) {
          const int m0 = m * kTile + rank * kHalf;
          const int n0 = p.v0 + n * kTile + rank * kHalf;
          if (m != kept) {
            if (keeps > 0 && !tc::mbar_wait(kempty_bar, (keeps - 1) & 1, s_abort)) break;
            fb = tc::mapa_shared(kfull_bar, 0);
            if (leader) tc::mbar_arrive_expect_tx(kfull_bar, 2 * keep * kSlot);
            for (int k = 0; k < keep; ++k) tc::tma_load_2d_pair(smem_base + k * kSlot, &tm_a, fb, k * kSlice, m0);
            kept = m;
            ++keeps;
          }
          for (int k = 0; k < p.k_slices; k += per) {
            if (k >= keep) {
              if ((dst = next_slot(kSlot, fb)) == 0) { ok = false; break; }
              tc::tma_load_2d_pair(dst, &tm_a, fb, k * kSlice, m0);
            }
            const int count = min(per, p.k_slices - k);
            if ((dst = next_slot(count * kSlot, fb)) == 0) { ok = false; break; }
            for (int i2 = 0; i2 < count; ++i2)
              tc::tma_load_2d_pair(dst + i2 * kSlot, &tm_b, fb, (k + i2) * kSlice, n0);
          }
        } else {
          const int m0 = m * kTile + rank * kHalf;
          const int n0 = n * p.n_cols;
          const int k0 = first_slice<ROLE>(p, at), k1 = last_slice<ROLE>(p, at);
          uint64_t next_parts = parts_of<ROLE>(p, at, k0);
          const int boxes1 = (n_first / 2 + 63) / 64, boxes2 = (n_second / 2 + 63) / 64;
          for (int k = k0; k < k1; ++k) {
            const uint64_t parts = next_parts;
            if (k + 1 < k1) next_parts = parts_of<ROLE>(p, at, k + 1);
            if ((dst = next_slot(kSlot, fb)) == 0) { ok = false; break; }
            const int block = S::A_MN ? m0 / kSlice : k;
            if (S::A_MN) {
              tc::tma_load_2d_pair(dst, &tm_a, fb, 0, 2 * block * p.g_rows + k * kSlice);
              tc::tma_load_2d_pair(dst + 8192, &tm_a, fb, 0, 2 * (block + 1) * p.g_rows + k * kSlice);
            } else {
              tc::tma_load_2d_pair(dst, &tm_a, fb, 0, 2 * block * p.g_rows + m0);
            }
            if (parts != 0) {
              // The second part, 32 rows of G at a time; zeros where there is none.
              if ((dst = next_slot(kSlot, fb)) == 0) { ok = false; break; }
              for (int i2 = 0; i2 < 4; ++i2) {
                const bool some = (parts >> (32 * rank + 8 * i2) & 0xff) != 0;
                const int row = S::A_MN ? (2 * (block + i2 / 2) + 1) * p.g_rows + k * kSlice + 32 * (i2 & 1)
                                        : (2 * block + 1) * p.g_rows + m0 + 32 * i2;
                tc::tma_load_2d_pair(dst + i2 * 4096, &tm_part, fb, 0, some ? row : p.g_all);
              }
            }
            const int k_row = k * kSlice + (ROLE == kGradQ ? p.v0 : 0);
            if ((dst = next_slot(boxes1 * 8192, fb)) == 0) { ok = false; break; }
            for (int b = 0; b < boxes1; ++b)
              tc::tma_load_2d_pair(dst + b * 8192, &tm_b, fb, n0 + rank * (n_first / 2) + 64 * b, k_row);
            if (n_second > 0) {
              if ((dst = next_slot(boxes2 * 8192, fb)) == 0) { ok = false; break; }
              for (int b = 0; b < boxes2; ++b)
                tc::tma_load_2d_pair(dst + b * 8192, &tm_b, fb, n0 + n_first + rank * (n_second / 2) + 64 * b, k_row);
            }
          }
        }
        advance<ROLE>(p, at);
      }
      // Both CTAs' loads complete on the even CTA's barriers: it waits for
      // the last phase of each before shared memory goes away.
      if (leader) {
        for (int64_t l = loads > ring ? loads - ring : 0; l < loads; ++l)
          quiet_wait(full_bar(static_cast<int>(l % ring)), static_cast<uint32_t>(l / ring) & 1);
        if (keeps > 0) quiet_wait(kfull_bar, (keeps - 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    // The whole warp walks the loop, so that descriptors and addresses stay in
    // uniform registers; one elected lane issues.
    if (leader) {
      const bool issuer = tc::elect_one();
      const uint64_t a_kind = S::A_MN ? tc::sw128_mnmajor_desc(0) : tc::sw128_kmajor_desc(0);
      const uint64_t b_kind = S::B_MN ? tc::sw128_mnmajor_desc(0) : tc::sw128_kmajor_desc(0);
      constexpr uint32_t kAStep = (S::A_MN ? 2048 : 32) >> 4, kBStep = (S::B_MN ? 2048 : 32) >> 4;
      int slot = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      uint32_t keeps = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, s_abort)) != 0;
      };
      // The next filled ring slot; false when a wait gave up.
      auto next_slot = [&](int& at) {
        if (!wait(full_bar(slot), phase)) return false;
        at = slot;
        if (++slot == ring) {
          slot = 0;
          phase ^= 1;
        }
        return true;
      };
      Place at = place_of<ROLE>(p, first);
      bool fresh = true;  // the queries changed
      for (int i = first; ok && i < last; i += step) {
        int k0 = 0, k1 = p.k_slices;
        uint64_t next_parts = 0;
        if (!S::LOGITS) {
          k0 = first_slice<ROLE>(p, at);
          k1 = last_slice<ROLE>(p, at);
          next_parts = parts_of<ROLE>(p, at, k0);
        }
        if (!wait(tempty_bar(acc), acc_phase ^ 1)) break;
        if (S::LOGITS) {
          if (fresh) {
            if (!wait(kfull_bar, keeps & 1)) break;
            ++keeps;
            fresh = false;
          }
        }
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kTile);
        for (int k = k0; k < k1; k += per) {
          int slot_a = -1, slot_l = -1, slot_b = -1, slot_c = -1;
          const bool streamed = !S::LOGITS || k >= keep;
          if (streamed && !next_slot(slot_a)) { ok = false; break; }
          const bool two = S::B_MN && next_parts != 0;  // G's second part
          if (S::B_MN && k + 1 < k1) next_parts = parts_of<ROLE>(p, at, k + 1);
          if (two && !next_slot(slot_l)) { ok = false; break; }
          if (!next_slot(slot_b)) { ok = false; break; }
          if (n_second > 0 && !next_slot(slot_c)) { ok = false; break; }
          tc::tc_fence_after();
          const uint32_t a_at = (streamed ? ring_base + slot_a * slot_bytes : smem_base + k * kSlot) >> 4;
          const uint64_t a_desc = a_kind + a_at;
          const uint64_t l_desc = a_kind + ((ring_base + slot_l * slot_bytes) >> 4);
          const uint64_t b_desc = b_kind + ((ring_base + slot_b * slot_bytes) >> 4);
          const uint64_t c_desc = b_kind + ((ring_base + slot_c * slot_bytes) >> 4);
          const uint32_t more = k > k0 ? 1u : 0u;
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_bf16_pair(d_tmem, a_desc + kk * kAStep, b_desc + kk * kBStep, p.idesc, kk > 0 ? 1u : more);
            if (S::LOGITS && per > 1 && k + 1 < k1) {  // the slot's second slice, against the next kept one
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_bf16_pair(d_tmem, a_desc + (kSlot >> 4) + kk * kAStep, b_desc + (kSlot >> 4) + kk * kBStep,
                                  p.idesc, 1u);
            }
            if (two) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_bf16_pair(d_tmem, l_desc + kk * kAStep, b_desc + kk * kBStep, p.idesc, 1u);
            }
            if (S::B_MN && n_second > 0) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_bf16_pair(d_tmem + kTile, a_desc + kk * kAStep, c_desc + kk * kBStep, p.idesc2,
                                  kk > 0 ? 1u : more);
              if (two) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  tc::mma_bf16_pair(d_tmem + kTile, l_desc + kk * kAStep, c_desc + kk * kBStep, p.idesc2, 1u);
              }
            }
            if (streamed) tc::mma_commit_pair_both(empty_bar(slot_a));
            if (two) tc::mma_commit_pair_both(empty_bar(slot_l));
            tc::mma_commit_pair_both(empty_bar(slot_b));
            if (S::B_MN && n_second > 0) tc::mma_commit_pair_both(empty_bar(slot_c));
          }
          __syncwarp();
        }
        if (!ok) break;
        if (issuer) tc::mma_commit_pair_both(tfull_bar(acc));
        const int m = at.m;
        advance<ROLE>(p, at);
        if (S::LOGITS && at.m != m) {
          fresh = true;
          if (issuer && i + 1 < last) tc::mma_commit_pair_both(kempty_bar);
        }
        __syncwarp();
        if (++acc == accs) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (issuer) tc::mma_commit_pair_both(done_bar);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int group = (warp - 2) >> 2;  // which 32-column blocks: group, group + 4, ...
    const int quarter = warp & 3;       // TMEM lanes this warp may access
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t out_buf = smem_base + kSlots * kSlot + (warp - 2) * kOutBuf;
    const int row_in_pair = rank * kHalf + quarter * 32 + lane;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool lost = false;  // a wait gave up: what remains is NaN
    int m_now = -1;
    // kStats / kWeights: the query's state.
    int target = -1;
    float run_base = -kInf, run_sum = 0.0f;
    float shift = -kInf, factor = 0.0f, at_target = 0.0f;
    auto flush = [&]() {  // kStats: this pair's (base, sum) of query tile m_now
      const int64_t q = static_cast<int64_t>(m_now) * kTile + row_in_pair;
      if (q < p.t) {
        const int slot = cluster - run_of(p.tiles, static_cast<int64_t>(m_now) * p.n_tiles, nclusters);
        p.part[q * p.lists + slot * kGroups + group] =
            make_float2(run_base, lost ? __int_as_float(0x7fc00000) : run_sum);
      }
    };
    Place place = place_of<ROLE>(p, first);
    // What the gradients are multiplied by at the end.
    const float final_scale =
        ROLE == kGradRows || (ROLE == kGradQ && p.direct) ? out_scale(p.row, p.scale) : 0.0f;
    for (int i = first; i < last; i += step) {
      const int m = place.m, n = place.n, split = place.split;
      advance<ROLE>(p, place);
      const int64_t row = static_cast<int64_t>(m) * kTile + row_in_pair;
      const int64_t row_warp = row - lane;
      if (S::LOGITS && m != m_now) {
        if (ROLE == kStats && m_now >= 0) flush();
        m_now = m;
        run_base = -kInf;
        run_sum = 0.0f;
        target = -1;
        factor = 0.0f;
        if (row < p.t) {
          const int64_t y = p.targets[row];
          const bool used = counts(y, p.ignore_index, p.v);
          if (used) target = static_cast<int>(y) - p.v0;
          if (ROLE == kWeights) {
            // G = factor * 2^(logit - lse) = +-2^(logit + shift); no row takes part
            // where lse is -inf.
            const float l = p.row.lse[row];
            factor = row_factor(p.row, used, row);
            shift = l == -kInf || factor == 0.0f ? -kInf : log2f(fabsf(factor)) - l * kLog2e;
            at_target = target_entry(p.row, row, factor);
          }
        }
      }
      if (S::LOGITS && BIAS) {
        // This warp's 64 biases come near while the tile is awaited (loss of 1000
        // x 500k x 128: 247 -> 227 us).
        const int64_t b = static_cast<int64_t>(p.v0) + n * kTile + group * 64 + lane * 32;
        if (lane < 2 && b < p.v) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.bias + b));
      }
      if (!lost && !__all_sync(0xffffffffu, tc::mbar_wait(tfull_bar(acc), acc_phase, s_abort))) lost = true;
      tc::tc_fence_after();
      if (ROLE == kStats) {
        // This warp's 64 columns.
        const int col = n * kTile + group * 64;
        const int left = static_cast<int>(p.v) - col;
        const bool some = row_warp < p.t && left > 0;
        const uint32_t at_tmem = lane_addr + static_cast<uint32_t>(acc * kTile + group * 64);
        // The columns are in registers: the accumulator is free.
        auto release = [&]() {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
        };
        auto take = [&](uint32_t (&v)[32], int first_col) {
          const int here = static_cast<int>(p.v) - first_col;
          if (BIAS) {
            add_bias(v, p.bias + first_col, here, p.c);
          } else if (here < 32) {
            leave_out_from(v, here);
          }
          // The target's logit stays out of the sum.
          const int at = target - first_col;
          if (at >= 0 && at < 32) leave_out(v, at);
          const float c = BIAS ? 1.0f : p.c;
          const float sum = block_sum(v, c, run_base);
          if (run_base != -kInf && sum < kRaise) {
            run_sum += sum;
          } else {
            const float top = largest(v) * c;
            if (top != -kInf) {  // something takes part (or is NaN)
              run_sum = run_sum * ex2(run_base - top) + block_sum(v, c, top);
              run_base = top;
            }
          }
        };
        if (some && lost) run_sum = __int_as_float(0x7fc00000);
        if (!some) {
          release();
        } else if (BIAS) {  // the bias's registers leave room for one half
          uint32_t v[32];
          __syncwarp();
          tc::tmem_ld_32x32b_x32(at_tmem, v);
          tc::tmem_ld_wait();
          take(v, col);
          __syncwarp();
          tc::tmem_ld_32x32b_x32(at_tmem + 32, v);
          tc::tmem_ld_wait();
          release();
          if (left > 32) take(v, col + 32);
        } else {
          uint32_t lo[32], hi[32];
          __syncwarp();
          tc::tmem_ld_32x32b_x32(at_tmem, lo);
          tc::tmem_ld_32x32b_x32(at_tmem + 32, hi);
          tc::tmem_ld_wait();
          release();
          take(lo, col);
          if (left > 32) take(hi, col + 32);
        }
        if (++acc == accs) {
          acc = 0;
          acc_phase ^= 1;
        }
        continue;
      }
      if (ROLE == kWeights) {
        // This warp's 64 columns, packed half by half.
        const int col = n * kTile + group * 64;  // within the piece
        const bool some = row_warp < p.g_rows && col < p.piece;
        const uint32_t at_tmem = lane_addr + static_cast<uint32_t>(acc * kTile + group * 64);
        auto release = [&]() {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
        };
        bool two = false;  // the block has a second part
        if (some) {
          // |G| of half `h` of the columns; past the base and left out: 0.
          auto entries = [&](uint32_t (&v)[32], int h) {
            __syncwarp();
            tc::tmem_ld_32x32b_x32(at_tmem + 32 * h, v);
            tc::tmem_ld_wait();
            if (lost) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
            }
            const int col_h = col + 32 * h;
            if (BIAS) {
              add_bias(v, p.bias + p.v0 + col_h, static_cast<int>(p.v) - p.v0 - col_h, p.c);
            } else if (p.piece - col_h < 32) {
              leave_out_from(v, p.piece - col_h);
            }
            const float c = BIAS ? 1.0f : p.c;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(ex2(fmaf(__uint_as_float(v[j]), c, shift)));
          };
          const uint32_t sign = factor < 0.0f ? 0x80008000u : 0;
          const int at = target - col;  // the target's place among the columns
          const bool mine = at >= 0 && at < 64;
          auto put = [&](uint32_t (&w)[32], float x) {  // x as the target's entry
            const uint32_t e = pack2<BF>(x, x);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (2 * j == at) w[j] = (w[j] & 0xffff0000u) | (e & 0xffffu);
              if (2 * j + 1 == at) w[j] = (w[j] & 0xffffu) | (e & 0xffff0000u);
            }
          };
          // A part leaves sixteen rows at a time, so that a buffer half as large as the
          // block takes rows of whole 128-byte lines (1-2% of a training step against
          // 64-byte ones).
          auto leave = [&](const uint32_t (&w)[32], int part) {
            const int g_row = (2 * (col / kSlice) + part) * p.g_rows + static_cast<int>(row_warp);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              stage_line(out_buf, lane, h, w);
              if (lane == 0) {
                tma_store(&tm_out, out_buf, 0, g_row + 16 * h);
                store_commit();
              }
            }
          };
          // A pass over the columns for each part, the second from the products again: the
          // same code, with no registers kept in between (with biases the first part's
          // entries, kept, made a piece of 333 x 50,021 x 100 take 45 us in place of 35).
#pragma unroll 1
          for (int part = 0; part == 0 || (part == 1 && two); ++part) {
            uint32_t w[32];
            float top = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t v[32];
              entries(v, h);
              if (part == 0) {
                top = max2(top, largest(v));
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  w[16 * h + j] = pack2<BF>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])) ^ sign;
              } else {
                // What the rounding took. The last columns are in registers: the accumulator is free.
                if (h == 1) release();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  const float a = __uint_as_float(v[2 * j]), b = __uint_as_float(v[2 * j + 1]);
                  const float2 r = widen2<BF>(pack2<BF>(a, b));
                  w[16 * h + j] = pack2<BF>(a - r.x, b - r.y) ^ sign;
                }
              }
            }
            if (part == 0) {
              if (mine) top = max2(top, fabsf(at_target));
              two = __any_sync(0xffffffffu, !(top <= kLarge * fabsf(factor)));
              if (!two) release();
            }
            if (mine) put(w, part == 0 ? at_target : at_target - rounded<BF>(at_target));
            leave(w, part);
          }
        } else {
          release();
        }
        if (lane == 0) {
          const int block = n * kGroups + group, rows32 = static_cast<int>(row_warp) / 32;
          p.parts_q[8 * (static_cast<int64_t>(block) * p.m_tiles + m) + rank * 4 + quarter] = two;
          if (row_warp < p.g_rows)
            p.parts_r[8 * (static_cast<int64_t>(n) * (p.g_rows / kSlice) + rows32 / 2) + group * 2 + (rows32 & 1)] = two;
        }
        if (++acc == accs) {
          acc = 0;
          acc_phase ^= 1;
        }
        continue;
      }
      const int64_t rows = ROLE == kGradRows ? p.piece : p.t;
      bool freed = false;
      if (row_warp < rows) {
        for (int b = group; b * 32 < p.n_cols; b += kGroups) {
          const int col = n * p.n_cols + b * 32;  // within the product
          const int cols = p.d;
          if (col >= cols) break;
          __syncwarp();
          uint32_t v[32];
          tc::tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * kTile + b * 32), v);
          tc::tmem_ld_wait();
          if ((b + kGroups) * 32 >= p.n_cols || col + kGroups * 32 >= cols) {
            // The warp's last columns are in registers: the accumulator is free.
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
            freed = true;
          }
          if (lost) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
          }
          if (ROLE == kGradQ && !p.direct) {
            // The split's slab, 16 fp32 columns at a time.
            const int slab_row = split * p.m_tiles * kTile + static_cast<int>(row_warp);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = v[16 * h + j];
              stage_row(out_buf, lane, w);
              if (lane == 0) {
                if (p.accumulate)
                  tma_add(&tm_out, out_buf, col + 16 * h, slab_row);
                else
                  tma_store(&tm_out, out_buf, col + 16 * h, slab_row);
                store_commit();
              }
            }
          }
          if (ROLE == kGradRows || (ROLE == kGradQ && p.direct)) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[j] = pack2<BF>(__uint_as_float(v[2 * j]) * final_scale, __uint_as_float(v[2 * j + 1]) * final_scale);
            stage_row(out_buf, lane, w);
            if (p.tma_out) {
              if (lane == 0) {
                tma_store(&tm_out, out_buf, col, p.out_row0 + static_cast<int>(row_warp));
                store_commit();
              }
            } else {
              store_staged(out_buf, lane, p.out + (p.out_row0 + row_warp) * p.ldo + col, p.ldo,
                           static_cast<int>(rows - row_warp), p.d - col);
              __syncwarp();
            }
          }
        }
      }
      if (!freed) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
      }
      if (++acc == accs) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (ROLE == kStats && m_now >= 0) flush();
    if (ROLE != kStats && lane == 0) store_wait();
  }

  if (warp == 1 && lane == 0) quiet_wait(done_bar, 0);
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 512);
  if (threadIdx.x == 0 && *s_abort) atomicOr(&g_xent_err, 1u);
}

// q . r of 16-bit values in fp32, a warp; rows start on 16-byte boundaries.
template <bool BF>
__device__ __forceinline__ float warp_dot(const uint16_t* q, const uint16_t* r, int d, int lane) {
  float s = 0.0f;
  for (int at = lane * 8; at < d; at += 256) {
    if (at + 8 <= d) {
      const uint4 a = *reinterpret_cast<const uint4*>(q + at);
      const uint4 b = *reinterpret_cast<const uint4*>(r + at);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w}, w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = widen2<BF>(u[j]), y = widen2<BF>(w[j]);
        s = fmaf(x.x, y.x, s);
        s = fmaf(x.y, y.y, s);
      }
    } else {
      for (int j = at; j < d; ++j) s = fmaf(widen2<BF>(q[j]).x, widen2<BF>(r[j]).x, s);
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  return s;
}

struct JoinArgs {
  const float2* part;
  int lists;           // pairs per query in part
  int n_tiles, pairs;  // base tiles, and how many CTA pairs shared the tiles
  int64_t tiles;
  const uint16_t *q, *rows;
  int64_t ldq, ldr, t, v;
  int d;
  float scale;
  const float* bias;
  const int64_t* targets;
  int64_t ignore_index;
  float *loss, *lse;
  int reduction;
  float *total, *divisor;
  unsigned* counter;
};

// One warp per query: joins the pairs' (base, sum), forms the target's logit
// and the loss. The last block to finish sums the losses, in 64 bits and a
// fixed order.
template <bool BF>
__global__ void __launch_bounds__(256) xent_join_kernel(const JoinArgs p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  wait_for_previous();
  let_next_start();
  if (row < p.t) {
    const int64_t m = row / kTile;
    const int used = kGroups * (run_of(p.tiles, (m + 1) * p.n_tiles - 1, p.pairs) - run_of(p.tiles, m * p.n_tiles, p.pairs) + 1);
    // The target's logit, before what does not depend on it.
    const int64_t y = p.targets[row];
    float zt = 0.0f;
    if (counts(y, p.ignore_index, p.v)) {
      zt = warp_dot<BF>(p.q + row * p.ldq, p.rows + y * p.ldr, p.d, lane) * p.scale;
      if (p.bias != nullptr) zt += bias2(p.bias[y]) * kLn2;
    }
    const float2* pr = p.part + row * p.lists;
    float top = -kInf;
    for (int i = lane; i < used; i += 32) top = fmaxf(top, pr[i].x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float base = top == -kInf ? 0.0f : top;
    float sum = 0.0f;
    for (int i = lane; i < used; i += 32) sum += pr[i].y * exp2f(pr[i].x - base);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float others = (base + log2f(sum)) * kLn2;  // -inf where no other row takes part
    float loss, lse = others;
    if (y == p.ignore_index) {
      loss = 0.0f;
    } else if (y < 0 || y >= p.v) {
      loss = __int_as_float(0x7fc00000);
    } else if (zt == -kInf) {  // the target is left out
      loss = sum == sum ? kInf : sum;
    } else {
      const float a = others - zt;
      const float tail = log1pf(expf(-fabsf(a)));
      loss = fmaxf(a, 0.0f) + tail + (a != a ? a : 0.0f);
      lse = fmaxf(others, zt) + tail;
    }
    if (lane == 0) {
      p.loss[row] = loss;
      p.lse[row] = lse;
    }
  }
  if (p.reduction == 0) return;
  __shared__ bool s_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.counter, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __shared__ double s_sum[8];
  __shared__ long long s_count[8];
  double sum = 0.0;
  long long count = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < p.t; i += 256) {
    const bool in = p.targets[i] != p.ignore_index;
    const float l = __ldcg(p.loss + i);
    sum += in ? l : 0.0f;
    count += in;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, s);
    count += __shfl_xor_sync(0xffffffffu, count, s);
  }
  if (lane == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_count[threadIdx.x >> 5] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) {
      sum += s_sum[w];
      count += s_count[w];
    }
    const double divisor = p.reduction == 2 ? static_cast<double>(count) : 1.0;
    p.total[0] = static_cast<float>(sum / divisor);
    p.divisor[0] = static_cast<float>(divisor);
  }
}

// One block: the largest finite |grad| of the queries that count.
__global__ void __launch_bounds__(1024) xent_top_kernel(const float* grad, const int64_t* targets,
                                                        int64_t ignore_index, int64_t t, int64_t v, float* out) {
  __shared__ float s_top[32];
  float top = 0.0f;
  wait_for_previous();
  let_next_start();
  for (int64_t i = threadIdx.x; i < t; i += 1024) {
    const float g = fabsf(grad[i]);
    if (g < kInf && counts(targets[i], ignore_index, v)) top = fmaxf(top, g);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) top = fmaxf(top, s_top[w]);
    out[0] = top;
  }
}

// Four values that nobody reads again.
__device__ __forceinline__ float4 load_once(const float4* p) {
  float4 r;
  asm volatile("ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
               : "l"(p)
               : "memory");
  return r;
}

struct GradQArgs {
  const float* slab;
  int splits;
  int64_t slab_rows, ld_slab, t;
  int d;
  RowGrad row;
  float scale;
  uint16_t* out;
  int64_t ldo;
  int rows_per_block;
};

// The sum of dq's slabs, scaled and rounded to the queries' type. A block takes
// rows_per_block rows, four columns per thread.
template <bool BF>
__global__ void __launch_bounds__(256) xent_grad_q_kernel(const GradQArgs p) {
  wait_for_previous();
  let_next_start();
  const int quads = (p.d + 3) / 4;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_block;
  const int work = p.rows_per_block * quads;
  const int64_t step = p.slab_rows * p.ld_slab / 4;
  const float f = out_scale(p.row, p.scale);
  for (int i = threadIdx.x; i < work; i += 256) {
    const int r_in = i / quads;
    const int64_t row = row0 + r_in;
    if (row >= p.t) break;
    const int col = (i - r_in * quads) * 4;
    const float4* s = reinterpret_cast<const float4*>(p.slab + row * p.ld_slab + col);
    float4 sum = load_once(s);
#pragma unroll 6
    for (int k = 1; k < p.splits; ++k) {
      const float4 w = load_once(s + k * step);
      sum.x += w.x;
      sum.y += w.y;
      sum.z += w.z;
      sum.w += w.w;
    }
    const uint32_t lo = pack2<BF>(sum.x * f, sum.y * f), hi = pack2<BF>(sum.z * f, sum.w * f);
    uint16_t* o = p.out + row * p.ldo + col;
    if (col + 4 <= p.d && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
      *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
    } else {
      o[0] = static_cast<uint16_t>(lo);
      if (col + 1 < p.d) o[1] = static_cast<uint16_t>(lo >> 16);
      if (col + 2 < p.d) o[2] = static_cast<uint16_t>(hi);
      if (col + 3 < p.d) o[3] = static_cast<uint16_t>(hi >> 16);
    }
  }
}

template <int ROLE>
cudaError_t launch_role(const CUtensorMap* maps, Args p, bool bf, int clusters, cudaStream_t stream) {
  p.next_m = clusters % p.m_tiles;
  p.next_n = clusters / p.m_tiles % p.n_tiles;
  p.next_split = clusters / p.m_tiles / p.n_tiles;
  constexpr bool kB = ROLE == kStats || ROLE == kWeights;
  const bool bias = kB && p.bias != nullptr;
  auto kern = bf ? (bias ? xent_gemm_kernel<ROLE, true, kB> : xent_gemm_kernel<ROLE, true, false>)
                 : (bias ? xent_gemm_kernel<ROLE, false, kB> : xent_gemm_kernel<ROLE, false, false>);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
  if (e != cudaSuccess) return e;
  return launch_after(kern, 2 * clusters, kThreads, kSmem, stream, maps[0], maps[1], maps[2], maps[3], p);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }
template <typename T>
T least(T a, T b) { return a < b ? a : b; }

// Pairs that share the forward's tiles. A multiple of the query tiles where
// that leaves at most a tenth idle: the runs of all query tiles then begin at
// the same base tiles, and the pairs that read the same base rows do so at the
// same time, from L2.
int stats_pairs(int64_t m_tiles, int64_t n_tiles, int clusters) {
  if (m_tiles * n_tiles <= clusters) return static_cast<int>(m_tiles * n_tiles);
  const int64_t even = clusters / m_tiles * m_tiles;
  return static_cast<int>(even * 10 >= clusters * 9 ? even : clusters);
}

// (base, sum) pairs per query: those of the most CTA pairs that share a query
// tile.
int stats_lists(int64_t m_tiles, int64_t n_tiles, int pairs) {
  int most = 1;
  for (int64_t m = 0; m < m_tiles; ++m) {
    const int n = run_of(m_tiles * n_tiles, (m + 1) * n_tiles - 1, pairs) - run_of(m_tiles * n_tiles, m * n_tiles, pairs) + 1;
    most = n > most ? n : most;
  }
  return most * kGroups;
}

// Tiles of the gradients' N side (d columns): equal widths up to 512, a
// multiple of 32.
struct GradTiles {
  int n_tiles, n_cols;
  explicit GradTiles(int d) {
    n_tiles = static_cast<int>(ceil_div(d, 2 * kTile));
    n_cols = static_cast<int>(align_up(ceil_div(d, n_tiles), 32));
  }
};

// Base tiles (of 256 columns) per piece of the backward. A piece's G is at
// most kPieceBytes, or two tiles (larger than L2: at d >= 256 the products take
// longer than G's way through HBM, and fewer pieces save more); among the sizes
// that fit, the one whose waves of logits and dr tiles take least, with a price
// per piece for its three launches and the adds into dq's slabs (about 16 us).
constexpr int64_t kPieceBytes = int64_t(256) << 20;
int64_t piece_tiles(int64_t t, int64_t v, int d, int clusters) {
  const GradTiles gt(d);
  const int64_t all = ceil_div(v, kTile), m_tiles = ceil_div(t, kTile);
  const int64_t per_tile = align_up(t, kSlice) * kTile * 4;  // bytes of G, both parts
  const int64_t fit = least(all, kPieceBytes / per_tile > 2 ? kPieceBytes / per_tile : int64_t(2));
  // Clocks of a tile of each product; its bytes of G cross HBM meanwhile.
  const double logits = ceil_div(d, kSlice) * 512.0, dr = ceil_div(t, kSlice) * 4.0 * gt.n_cols;
  auto cost = [&](int64_t tiles) {
    return 30000.0 + logits * ceil_div(tiles * m_tiles, clusters) + dr * ceil_div(tiles * gt.n_tiles, clusters);
  };
  int64_t best = fit;
  double best_cost = 0;
  // Sizes that fill whole waves, and equal divisions of the base.
  auto consider = [&](int64_t tiles) {
    if (tiles < 1 || tiles > fit) return;
    const int64_t rest = all % tiles;
    const double c = (all / tiles) * cost(tiles) + (rest > 0 ? cost(rest) : 0);
    if (best_cost == 0 || c < best_cost) {
      best_cost = c;
      best = tiles;
    }
  };
  for (int64_t n = ceil_div(all, fit); n <= ceil_div(all, fit) + 8; ++n) consider(ceil_div(all, n));
  for (int64_t w = 1; w <= 16; ++w) consider(w * clusters / gt.n_tiles);
  return best;
}

int grad_q_splits(int64_t m_tiles, int64_t n_tiles, int64_t slices, int clusters) {
  int64_t s = clusters / (m_tiles * n_tiles);
  if (s < 1) s = 1;
  if (s > slices) s = slices;
  return static_cast<int>(s);
}

struct Carve {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used = align_up(used + count * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};

struct ForwardPlan {
  int m_tiles, n_tiles, pairs, lists;
  float2* part;
  unsigned* counter;
  int64_t bytes;
  ForwardPlan(void* ws, int64_t t, int64_t v, int clusters) {
    m_tiles = static_cast<int>(ceil_div(t, kTile));
    n_tiles = static_cast<int>(ceil_div(v, kTile));
    pairs = stats_pairs(m_tiles, n_tiles, clusters);
    lists = stats_lists(m_tiles, n_tiles, pairs);
    Carve c{static_cast<char*>(ws)};
    part = c.take<float2>(t * lists);
    counter = c.take<unsigned>(1);
    bytes = c.used;
  }
};

struct BackwardPlan {
  GradTiles gt;
  int m_tiles, q_splits, g_rows;
  int64_t piece, slab_rows, ld_slab;  // columns of a piece
  float *top, *slab;
  uint16_t* g;
  uint8_t *parts_q, *parts_r;  // a byte per block of 32 rows x 64 columns of G
  int64_t bytes;
  BackwardPlan(void* ws, int64_t t, int64_t v, int d, int clusters) : gt(d) {
    m_tiles = static_cast<int>(ceil_div(t, kTile));
    piece = piece_tiles(t, v, d, clusters) * kTile;
    q_splits = grad_q_splits(m_tiles, gt.n_tiles, least(piece, v) / kSlice + 1, clusters);
    slab_rows = static_cast<int64_t>(m_tiles) * kTile;
    ld_slab = static_cast<int64_t>(gt.n_tiles) * gt.n_cols;
    Carve c{static_cast<char*>(ws)};
    top = c.take<float>(1);
    slab = c.take<float>(q_splits * slab_rows * ld_slab);
    g_rows = static_cast<int>(align_up(t, kSlice));
    g = c.take<uint16_t>(2 * piece * g_rows);
    parts_q = c.take<uint8_t>(piece / kSlice * m_tiles * 8);
    parts_r = c.take<uint8_t>(piece / kTile * (g_rows / kSlice) * 8);
    bytes = c.used;
  }
};

Args common_args(const XentProblem& x) {
  Args p = {};
  p.t = x.t;
  p.v = x.v;
  p.d = x.d;
  p.c = x.scale * kLog2e;
  p.scale = x.scale;
  p.bias = x.bias;
  p.targets = x.targets;
  p.ignore_index = x.ignore_index;
  return p;
}

// The logits' tiles: queries x n_tiles base tiles.
void logits_args(Args& p, bool bf, int m_tiles, int n_tiles) {
  p.m_tiles = m_tiles;
  p.n_tiles = n_tiles;
  p.tiles = m_tiles * n_tiles;
  p.n_cols = kTile;
  p.k_slices = static_cast<int>(ceil_div(p.d, kSlice));
  p.keep = least(p.k_slices, kKeep);
  // Two slices per slot where the ring still holds three: half the waits and
  // commits of a short tile.
  p.per_slot = p.k_slices <= 6 ? 2 : 1;
  p.idesc = p.idesc2 = tc::idesc_16(bf, false, false, kTile, kTile);
}

// A gradient's tiles.
void grad_args(Args& p, const GradTiles& gt, bool bf, bool a_mn, int m_tiles, int64_t k, int splits) {
  p.m_tiles = m_tiles;
  p.n_tiles = gt.n_tiles;
  p.n_cols = gt.n_cols;
  p.k_slices = static_cast<int>(ceil_div(k, kSlice));
  p.per_split = static_cast<int>(ceil_div(p.k_slices, splits));
  p.tiles = m_tiles * gt.n_tiles * static_cast<int>(ceil_div(p.k_slices, p.per_split));
  const int first = least(gt.n_cols, kTile);
  p.idesc = tc::idesc_16(bf, a_mn, true, kTile, first);
  p.idesc2 = tc::idesc_16(bf, a_mn, true, kTile, gt.n_cols > kTile ? gt.n_cols - first : first);
}

}  // namespace

int64_t xent_forward_workspace(int64_t t, int64_t v, int clusters) { return ForwardPlan(nullptr, t, v, clusters).bytes; }

int64_t xent_backward_workspace(int64_t t, int64_t v, int d, int clusters) {
  return BackwardPlan(nullptr, t, v, d, clusters).bytes;
}

cudaError_t launch_xent_forward(const XentProblem& x, float* loss, float* lse, int reduction, float* total,
                                float* divisor, void* ws, int clusters, cudaStream_t stream, int* launches) {
  const bool bf = x.type == kElemBf16;
  const ForwardPlan plan(ws, x.t, x.v, clusters);
  Args p = common_args(x);
  logits_args(p, bf, plan.m_tiles, plan.n_tiles);
  p.part = plan.part;
  p.lists = plan.lists;
  p.counter = plan.counter;
  CUtensorMap maps[4];
  cudaError_t e = encode_rows_map(&maps[0], x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kHalf, 128);
  if (e == cudaSuccess) e = encode_rows_map(&maps[1], x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kHalf, 128);
  maps[2] = maps[3] = maps[0];  // not used
  if (e == cudaSuccess) e = launch_role<kStats>(maps, p, bf, plan.pairs, stream);
  if (e != cudaSuccess) return e;
  JoinArgs j = {};
  j.part = plan.part;
  j.lists = plan.lists;
  j.n_tiles = plan.n_tiles;
  j.pairs = plan.pairs;
  j.tiles = p.tiles;
  j.q = static_cast<const uint16_t*>(x.q);
  j.rows = static_cast<const uint16_t*>(x.rows);
  j.ldq = x.ldq;
  j.ldr = x.ldr;
  j.t = x.t;
  j.v = x.v;
  j.d = x.d;
  j.scale = x.scale;
  j.bias = x.bias;
  j.targets = x.targets;
  j.ignore_index = x.ignore_index;
  j.loss = loss;
  j.lse = lse;
  j.reduction = reduction;
  j.total = total;
  j.divisor = divisor;
  j.counter = plan.counter;
  auto join = bf ? xent_join_kernel<true> : xent_join_kernel<false>;
  *launches = 2;
  return launch_after(join, ceil_div(x.t, 8), 256, 0, stream, j);
}

cudaError_t launch_xent_backward(const XentProblem& x, const float* loss, const float* lse, const float* grad,
                                 int grad_stride, const float* divisor, void* dq, int64_t lddq, void* drows,
                                 int64_t lddr, void* ws, int clusters, cudaStream_t stream, int* launches) {
  const bool bf = x.type == kElemBf16;
  const BackwardPlan plan(ws, x.t, x.v, x.d, clusters);
  cudaError_t e;
  RowGrad row = {loss, lse, grad, grad, divisor, grad_stride, bf ? 1.0f : 16384.0f};
  if (grad_stride != 0) {
    e = launch_after(xent_top_kernel, 1, 1024, 0, stream, grad, x.targets, x.ignore_index, x.t, x.v, plan.top);
    if (e != cudaSuccess) return e;
    ++*launches;
    row.top = plan.top;
  }
  Args base = common_args(x);
  base.row = row;

  CUtensorMap q_k, rows_k, q_mn, rows_mn, slab, dr, dq_map;
  e = encode_rows_map(&q_k, x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kHalf, 128);
  if (e == cudaSuccess) e = encode_rows_map(&rows_k, x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kHalf, 128);
  // MN-major operands: boxes of 64 columns by 64 rows.
  if (e == cudaSuccess) e = encode_rows_map(&rows_mn, x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kSlice, 128);
  if (e == cudaSuccess) e = encode_rows_map(&q_mn, x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kSlice, 128);
  // Stores: an epilogue warp's 32 rows of 64 bytes.
  if (e == cudaSuccess)
    e = encode_rows_map(&slab, kElemF32, plan.slab, plan.ld_slab, plan.q_splits * plan.slab_rows, plan.ld_slab * 4, 16,
                        32, 64);
  // TMA stores whole 16-byte pieces: a row that ends inside one would take what
  // lies behind it along.
  auto by_tma = [&](const void* p, int64_t ld) {
    return p != nullptr && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && x.d % 8 == 0;
  };
  const bool dr_tma = by_tma(drows, lddr), dq_tma = by_tma(dq, lddq);
  dr = dq_map = slab;
  if (e == cudaSuccess && dr_tma) e = encode_rows_map(&dr, x.type, drows, x.d, x.v, lddr * 2, 32, 32, 64);
  if (e == cudaSuccess && dq_tma) e = encode_rows_map(&dq_map, x.type, dq, x.d, x.t, lddq * 2, 32, 32, 64);
  if (e != cudaSuccess) return e;
  base.g_rows = plan.g_rows;
  base.parts_q = plan.parts_q;
  base.parts_r = plan.parts_r;
  int splits_used = 0;
  bool direct = false;
  for (int64_t v0 = 0; v0 < x.v; v0 += plan.piece) {
    const int64_t piece = least(plan.piece, x.v - v0);
    const int piece_n = static_cast<int>(ceil_div(piece, kTile));
    base.v0 = static_cast<int>(v0);
    base.piece = static_cast<int>(piece);
    CUtensorMap g_k, g_mn, g_out, g_part;
    const int64_t g_all = 2 * ceil_div(piece, kSlice) * plan.g_rows;
    if (g_all > 0x7fffff00) return cudaErrorInvalidValue;  // TMA coordinates are 32-bit (a G of 275 GB)
    e = encode_rows_map(&g_k, x.type, plan.g, kSlice, g_all, kSlice * 2, kSlice, kHalf, 128);
    if (e == cudaSuccess) e = encode_rows_map(&g_mn, x.type, plan.g, kSlice, g_all, kSlice * 2, kSlice, kSlice, 128);
    if (e == cudaSuccess) e = encode_rows_map(&g_out, x.type, plan.g, kSlice, g_all, kSlice * 2, kSlice, 16, 128);
    if (e == cudaSuccess) e = encode_rows_map(&g_part, x.type, plan.g, kSlice, g_all, kSlice * 2, kSlice, 32, 128);
    if (e != cudaSuccess) return e;
    base.g_all = static_cast<int>(g_all);
    Args p = base;
    logits_args(p, bf, plan.m_tiles, piece_n);
    CUtensorMap maps[4] = {q_k, rows_k, g_out, g_out};
    if ((e = launch_role<kWeights>(maps, p, bf, least(clusters, p.tiles), stream)) != cudaSuccess) return e;
    ++*launches;
    if (dq != nullptr) {
      p = base;
      // Later pieces use no slab that the first did not write.
      grad_args(p, plan.gt, bf, false, plan.m_tiles, piece, splits_used > 0 ? splits_used : plan.q_splits);
      if (splits_used == 0) splits_used = p.tiles / (p.m_tiles * p.n_tiles);
      p.accumulate = v0 > 0;
      p.direct = splits_used == 1 && piece == x.v;
      p.out = static_cast<uint16_t*>(dq);
      p.ldo = lddq;
      p.tma_out = dq_tma;
      direct = p.direct != 0;
      CUtensorMap maps_q[4] = {g_k, rows_mn, direct ? dq_map : slab, g_part};
      if ((e = launch_role<kGradQ>(maps_q, p, bf, least(clusters, p.tiles), stream)) != cudaSuccess) return e;
      ++*launches;
    }
    if (drows != nullptr) {
      p = base;
      grad_args(p, plan.gt, bf, true, piece_n, x.t, 1);
      p.out = static_cast<uint16_t*>(drows);
      p.ldo = lddr;
      p.out_row0 = static_cast<int>(v0);
      p.tma_out = dr_tma;
      CUtensorMap maps_r[4] = {g_mn, q_mn, dr, g_part};
      if ((e = launch_role<kGradRows>(maps_r, p, bf, least(clusters, p.tiles), stream)) != cudaSuccess) return e;
      ++*launches;
    }
  }
  if (dq != nullptr && !direct) {
    const int quads = static_cast<int>(ceil_div(x.d, 4));
    const int rows_per_block = quads >= 256 ? 1 : 256 / quads;
    GradQArgs a = {plan.slab, splits_used, plan.slab_rows, plan.ld_slab, x.t, x.d, row, x.scale,
                   static_cast<uint16_t*>(dq), lddq, rows_per_block};
    e = launch_after(bf ? xent_grad_q_kernel<true> : xent_grad_q_kernel<false>, ceil_div(x.t, rows_per_block), 256, 0,
                     stream, a);
    ++*launches;
  }
  return e;
}

cudaError_t take_xent_error(cudaStream_t stream, unsigned* out) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_xent_err, sizeof(unsigned), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *out == 0) return e;
  const unsigned zero = 0;
  e = cudaMemcpyToSymbolAsync(g_xent_err, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, stream);
  return e == cudaSuccess ? cudaStreamSynchronize(stream) : e;
}

}  // namespace px
