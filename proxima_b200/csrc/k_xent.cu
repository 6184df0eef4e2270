// Softmax cross entropy of queries over a whole base, and its gradient,
// without the t x v matrix of logits:
//     z_ij = scale * q_i . r_j + bias_j
//     loss_i = log sum_j exp z_ij - z_i,y(i)
//     G_ij = g_i (exp(z_ij - lse_i) - [j = y(i)]),  dq = scale * G r,  dr = scale * G^T q
//
// Forward: one pass over the products, whose epilogue keeps a running maximum
// and sum per query and split of the base; a second kernel joins the splits.
// The target's own logit stays out of the sum, so the loss is
//     softplus(log sum_{j != y} exp z_ij - z_iy),
// which does not cancel when the target holds nearly all of the softmax.
//
// Backward: the base is taken in pieces of columns. For each piece the
// products are computed again, their epilogue writes the piece of G in the
// operands' 16-bit type (a buffer of at most 64 MB, so it is read back from
// L2), and two more products read it: dq accumulates over the pieces in fp32
// slabs (one per split of the piece, added to in the same order every time,
// so results do not change from run to run), dr is complete per piece.
// G's rounding to 16 bits is the one rounding beside the outputs': relative
// 2^-9 (bf16) or 2^-12 (fp16) of each entry, as the outputs' own. Entries are
// relative to the largest |g_i|, times 2^14 for fp16, whose smallest normal
// would otherwise lie above the probabilities of a large base.
//
// All three products are one kernel, instantiated per role: CTA pairs
// (tcgen05.mma cta_group::2, kind::f16), 256 x N tiles with N <= 256, a
// 6-stage TMA ring of 64-deep slices, two TMEM accumulators, the epilogue
// (8 warps per CTA) overlapping the next tile. The three read their operands
// as they lie: G^T, the base as dq's right operand and the queries as dr's are
// MN-major tiles, so nothing is transposed in memory.
//
// Bound: the tensor pipe for d >= 256 or so (2 t v d operations forward, three
// times that backward, of which the logits again are the price of not keeping
// them); the forward at small d by the exponentials (one per logit).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "px_rows.h"
#include "px_tc.cuh"

namespace px {

namespace {

// Set when a bounded wait gave up (px_rows_status_device reads and clears it).
__device__ unsigned g_xent_err;

constexpr int kHalf = 128;   // M rows per CTA (TMEM lanes)
constexpr int kTile = 256;   // M rows per pair, and the most N columns
constexpr int kSlice = 64;   // K values per slice: 128 bytes
constexpr int kStages = 6;
constexpr int kOperand = kHalf * 128;  // 16 KB
constexpr int kStage = 2 * kOperand;
constexpr int kThreads = 64 + 256;
constexpr int kBars = 2 * kStages + 2 + 2 + 1;
constexpr size_t kSmem = 1024 + kStages * kStage + kBars * 8 + 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

enum Role { kStats, kWeights, kGradQ, kGradRows };

template <int ROLE> struct Shape {
  static constexpr bool A_MN = ROLE == kGradRows;
  static constexpr bool B_MN = ROLE == kGradQ || ROLE == kGradRows;
};

struct Args {
  int64_t t, v;
  int d;
  int m_tiles, n_tiles;  // tiles of the product (kStats: n_tiles base tiles in all)
  int splits, per_split; // kStats: base tiles per split; kGradQ: K slices per split
  int n_items;
  int n_cols;            // N of a tile
  int k_slices;
  int64_t v0;            // first base row of the piece
  int64_t piece;         // its columns
  uint32_t idesc;
  float c;               // scale * log2(e)
  const float* bias;
  const int64_t* targets;
  int64_t ignore_index;
  float2* part;          // kStats: [t][splits * 2] (max, sum), log2 units
  float* target_z;       // kStats: [t] the target's logit, log2 units
  const float* lse2;     // kWeights: [t], log2 units
  const float* row_factor;  // kWeights: [t]
  const float* target_g;    // kWeights: [t] the target's entry before the row factor
  void* g;               // kWeights: [t][ldg]
  int64_t ldg;
  float* slab;           // kGradQ: [splits][m_tiles * 256][ld_slab]
  int64_t ld_slab;
  int accumulate;
  const float* out_scale;  // kGradRows: one value
  void* out;             // kGradRows: rows v0 .. of the base's gradient
  int64_t ldo;
  int vec_out;
};

// Item -> the tiles a pair computes: M tile, first N tile and their count, K
// slices [k0, k1).
struct Item {
  int m, n, n_end, k0, k1, split;
};

template <int ROLE>
__device__ __forceinline__ Item item_of(const Args& p, int i) {
  Item it;
  it.k0 = 0;
  it.k1 = p.k_slices;
  it.split = 0;
  it.m = i % p.m_tiles;
  const int rest = i / p.m_tiles;
  if (ROLE == kStats) {
    it.split = rest;
    it.n = rest * p.per_split;
    it.n_end = min(p.n_tiles, it.n + p.per_split);
  } else if (ROLE == kGradQ) {
    it.n = rest % p.n_tiles;
    it.n_end = it.n + 1;
    it.split = rest / p.n_tiles;
    it.k0 = it.split * p.per_split;
    it.k1 = min(p.k_slices, it.k0 + p.per_split);
  } else {
    it.n = rest;
    it.n_end = it.n + 1;
  }
  return it;
}

__device__ __forceinline__ void quiet_wait(uint32_t bar, uint32_t parity) {
  int dummy = 0;
  tc::mbar_wait(bar, parity, &dummy);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
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

// Logits of 32 columns in log2 units: c * (q . r) + bias * log2(e). Columns
// past the base, and base rows left out by a bias of -inf, are -inf whatever
// their product.
template <bool BIAS>
__device__ __forceinline__ void logits32(const uint32_t (&v)[32], const Args& p, int64_t col0, float (&z)[32]) {
  const bool whole = col0 + 32 <= p.v;
  if (BIAS) {
    if (whole) {
      const float4* b4 = reinterpret_cast<const float4*>(p.bias + col0);
#pragma unroll
      for (int j4 = 0; j4 < 8; ++j4) {
        const float4 b = __ldg(b4 + j4);
        const float w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int h = 0; h < 4; ++h)
          z[4 * j4 + h] = w[h] == -kInf ? -kInf : fmaf(__uint_as_float(v[4 * j4 + h]), p.c, w[h] * kLog2e);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float b = col0 + j < p.v ? __ldg(p.bias + col0 + j) : -kInf;
        z[j] = b == -kInf ? -kInf : fmaf(__uint_as_float(v[j]), p.c, b * kLog2e);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j] = whole || col0 + j < p.v ? __uint_as_float(v[j]) * p.c : -kInf;
  }
}

template <int ROLE, bool BF, bool BIAS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
xent_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const Args p) {
  using S = Shape<ROLE>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * kStage);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t smem_base = tc::smem_addr(smem);
  auto full_bar = [&](int s) { return tc::smem_addr(&bars[s]); };
  auto empty_bar = [&](int s) { return tc::smem_addr(&bars[kStages + s]); };
  auto tfull_bar = [&](int a) { return tc::smem_addr(&bars[2 * kStages + a]); };
  auto tempty_bar = [&](int a) { return tc::smem_addr(&bars[2 * kStages + 2 + a]); };
  const uint32_t done_bar = tc::smem_addr(&bars[2 * kStages + 4]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(tfull_bar(a), 1);
      tc::mbar_init(tempty_bar(a), 16);
    }
    tc::mbar_init(done_bar, 1);
    *s_abort = 0;
    tc::fence_mbarrier_init_cluster();
  }
  if (warp == 0 && lane == 0) {
    tc::prefetch_tmap(&tm_a);
    tc::prefetch_tmap(&tm_b);
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
  const int cluster = static_cast<int>(tc::cluster_id_x());
  const int nclusters = static_cast<int>(tc::nclusters_x());
  // Boxes of 64 columns that hold this CTA's half of an MN-major B tile.
  const int b_boxes = S::B_MN ? (p.n_cols / 2 + 63) / 64 : 1;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t bytes = kOperand + (S::B_MN ? b_boxes * 8192 : kOperand);
      int64_t loads = 0;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = cluster; ok && i < p.n_items; i += nclusters) {
        const Item it = item_of<ROLE>(p, i);
        const int m0 = it.m * kTile + static_cast<int>(rank) * kHalf;
        for (int n = it.n; ok && n < it.n_end; ++n) {
          const int n0 = n * p.n_cols + static_cast<int>(rank) * (p.n_cols / 2);
          for (int k = it.k0; k < it.k1; ++k) {
            if (!tc::mbar_wait(empty_bar(stage), phase ^ 1, s_abort)) {
              ok = false;
              break;
            }
            const uint32_t a_dst = smem_base + stage * kStage;
            const uint32_t b_dst = a_dst + kOperand;
            const uint32_t fb = tc::mapa_shared(full_bar(stage), 0);
            if (leader) tc::mbar_arrive_expect_tx(full_bar(stage), 2 * bytes);
            if (S::A_MN) {
              tc::tma_load_2d_pair(a_dst, &tm_a, fb, m0, k * kSlice);
              tc::tma_load_2d_pair(a_dst + 8192, &tm_a, fb, m0 + 64, k * kSlice);
            } else {
              tc::tma_load_2d_pair(a_dst, &tm_a, fb, k * kSlice, m0);
            }
            if (S::B_MN) {
              const int k_row = k * kSlice + (ROLE == kGradQ ? static_cast<int>(p.v0) : 0);
              for (int b = 0; b < b_boxes; ++b)
                tc::tma_load_2d_pair(b_dst + b * 8192, &tm_b, fb, n0 + 64 * b, k_row);
            } else {
              tc::tma_load_2d_pair(b_dst, &tm_b, fb, k * kSlice, static_cast<int>(p.v0) + n0);
            }
            ++loads;
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
      }
      // Both CTAs' loads complete on the even CTA's barriers: it waits for
      // the last phase of each before shared memory goes away.
      if (leader)
        for (int64_t l = loads > kStages ? loads - kStages : 0; l < loads; ++l)
          quiet_wait(full_bar(static_cast<int>(l % kStages)), static_cast<uint32_t>(l / kStages) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    if (leader && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int i = cluster; ok && i < p.n_items; i += nclusters) {
        const Item it = item_of<ROLE>(p, i);
        for (int n = it.n; ok && n < it.n_end; ++n) {
          if (!tc::mbar_wait(tempty_bar(acc), acc_phase ^ 1, s_abort)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kTile);
          for (int k = it.k0; k < it.k1; ++k) {
            if (!tc::mbar_wait(full_bar(stage), phase, s_abort)) {
              ok = false;
              break;
            }
            tc::tc_fence_after();
            const uint32_t a_addr = smem_base + stage * kStage;
            const uint32_t b_addr = a_addr + kOperand;
            const uint64_t a_desc = S::A_MN ? tc::sw128_mnmajor_desc(a_addr) : tc::sw128_kmajor_desc(a_addr);
            const uint64_t b_desc = S::B_MN ? tc::sw128_mnmajor_desc(b_addr) : tc::sw128_kmajor_desc(b_addr);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t a_off = static_cast<uint64_t>(kk * (S::A_MN ? 2048 : 32)) >> 4;
              const uint64_t b_off = static_cast<uint64_t>(kk * (S::B_MN ? 2048 : 32)) >> 4;
              tc::mma_bf16_pair(d_tmem, a_desc + a_off, b_desc + b_off, p.idesc, (k > it.k0 || kk > 0) ? 1u : 0u);
            }
            tc::mma_commit_pair_both(empty_bar(stage));
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          tc::mma_commit_pair_both(tfull_bar(acc));
          if (++acc == 2) {
            acc = 0;
            acc_phase ^= 1;
          }
        }
      }
      tc::mma_commit_pair_both(done_bar);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int half = (warp - 2) >> 2;  // which alternate blocks of 32 columns
    const int quarter = warp & 3;      // TMEM lanes this warp may access
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const float nan = __int_as_float(0x7fc00000);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool lost = false;  // a wait gave up: what remains is NaN
    for (int i = cluster; i < p.n_items; i += nclusters) {
      const Item it = item_of<ROLE>(p, i);
      const int64_t m_warp = static_cast<int64_t>(it.m) * kTile + rank * kHalf + quarter * 32;
      const int64_t m = m_warp + lane;
      const bool live = ROLE == kGradRows ? m < p.piece : m < p.t;
      int64_t target = -1;
      float run_max = -kInf, run_sum = 0.0f;
      float lse2 = 0.0f, factor = 0.0f, target_g = 0.0f;
      float out_scale = 0.0f;
      if (ROLE == kStats || ROLE == kWeights) {
        if (live) target = __ldg(p.targets + m);
        if (target == p.ignore_index) target = -1;
      }
      if (ROLE == kWeights && live) {
        lse2 = __ldg(p.lse2 + m);
        factor = __ldg(p.row_factor + m);
        target_g = __ldg(p.target_g + m);
      }
      if (ROLE == kGradRows) out_scale = __ldg(p.out_scale);
      for (int n = it.n; n < it.n_end; ++n) {
        if (!lost && !__all_sync(0xffffffffu, tc::mbar_wait(tfull_bar(acc), acc_phase, s_abort))) lost = true;
        tc::tc_fence_after();
        const int64_t n0 = static_cast<int64_t>(n) * p.n_cols;
        if (m_warp < (ROLE == kGradRows ? p.piece : p.t)) {
          for (int b = half; b * 32 < p.n_cols; b += 2) {
            const int64_t col = n0 + b * 32;  // within the product
            if (ROLE == kStats && col >= p.v) break;
            if (ROLE == kWeights && col >= p.piece) break;
            if (ROLE == kGradRows && col >= p.d) break;
            __syncwarp();
            uint32_t v[32];
            tc::tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * kTile + b * 32), v);
            tc::tmem_ld_wait();
            if (lost) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = 0x7fc00000u;
            }
            if (ROLE == kStats) {
              float z[32];
              logits32<BIAS>(v, p, col, z);
              const int64_t at = target - col;
              if (at >= 0 && at < 32) {  // the target's logit leaves the sum
                float zt = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j == at) {
                    zt = z[j];
                    z[j] = -kInf;
                  }
                p.target_z[m] = zt;
              }
              float top = run_max;
#pragma unroll
              for (int j = 0; j < 32; ++j) top = fmaxf(top, z[j]);
              const float base = top == -kInf ? 0.0f : top;
              float sum = run_sum * ex2(run_max - base);
              float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int j = 0; j < 32; ++j) s[j & 3] += ex2(z[j] - base);
              run_sum = sum + ((s[0] + s[1]) + (s[2] + s[3]));
              run_max = top;
            }
            if (ROLE == kWeights) {
              float z[32];
              logits32<BIAS>(v, p, p.v0 + col, z);
#pragma unroll
              for (int j = 0; j < 32; ++j) z[j] = factor == 0.0f ? 0.0f : ex2(z[j] - lse2) * factor;
              const int64_t at = target - (p.v0 + col);
              if (at >= 0 && at < 32) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (j == at) z[j] = factor == 0.0f ? 0.0f : target_g * factor;
              }
              if (live) {
                uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.g) + m * p.ldg + col);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  uint4 w;
                  w.x = pack2<BF>(z[8 * j], z[8 * j + 1]);
                  w.y = pack2<BF>(z[8 * j + 2], z[8 * j + 3]);
                  w.z = pack2<BF>(z[8 * j + 4], z[8 * j + 5]);
                  w.w = pack2<BF>(z[8 * j + 6], z[8 * j + 7]);
                  o[j] = w;
                }
              }
            }
            if (ROLE == kGradQ && live) {
              float4* o = reinterpret_cast<float4*>(
                  p.slab + (static_cast<int64_t>(it.split) * p.m_tiles * kTile + m) * p.ld_slab + col);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float4 w = p.accumulate ? o[j] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                w.x += __uint_as_float(v[4 * j]);
                w.y += __uint_as_float(v[4 * j + 1]);
                w.z += __uint_as_float(v[4 * j + 2]);
                w.w += __uint_as_float(v[4 * j + 3]);
                o[j] = w;
              }
            }
            if (ROLE == kGradRows && live) {
              uint16_t* o = static_cast<uint16_t*>(p.out) + (p.v0 + m) * p.ldo + col;
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j)
                w[j] = pack2<BF>(__uint_as_float(v[2 * j]) * out_scale, __uint_as_float(v[2 * j + 1]) * out_scale);
              if (p.vec_out && col + 32 <= p.d) {
                uint4* o4 = reinterpret_cast<uint4*>(o);
#pragma unroll
                for (int j = 0; j < 4; ++j) __stcs(o4 + j, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]));
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  if (col + 2 * j < p.d) o[2 * j] = static_cast<uint16_t>(w[j]);
                  if (col + 2 * j + 1 < p.d) o[2 * j + 1] = static_cast<uint16_t>(w[j] >> 16);
                }
              }
            }
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (ROLE == kStats && live) {
        if (lost) run_sum = nan;
        p.part[(m * p.splits + it.split) * 2 + half] = make_float2(run_max, run_sum);
      }
    }
  }

  if (warp == 1 && lane == 0) quiet_wait(done_bar, 0);
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 512);
  if (threadIdx.x == 0 && *s_abort) atomicOr(&g_xent_err, 1u);
}

// One warp per query: joins the splits' (max, sum) and forms the loss.
__global__ void __launch_bounds__(256) xent_join_kernel(const float2* __restrict__ part, int per_row,
                                                        const float* __restrict__ target_z,
                                                        const int64_t* __restrict__ targets, int64_t ignore_index,
                                                        int64_t t, int64_t v, float* __restrict__ loss,
                                                        float* __restrict__ lse) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= t) return;
  const int lane = threadIdx.x & 31;
  const float2* pr = part + row * per_row;
  float top = -kInf;
  for (int i = lane; i < per_row; i += 32) top = fmaxf(top, pr[i].x);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  const float base = top == -kInf ? 0.0f : top;
  float sum = 0.0f;
  for (int i = lane; i < per_row; i += 32) sum += pr[i].y * exp2f(pr[i].x - base);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if (lane != 0) return;
  const int64_t y = targets[row];
  const float others = (base + log2f(sum)) * kLn2;  // -inf where no other row takes part
  if (y == ignore_index) {
    // target_z was not written, and nothing left the sum.
    loss[row] = 0.0f;
    lse[row] = others;
  } else if (y < 0 || y >= v) {
    loss[row] = __int_as_float(0x7fc00000);
    lse[row] = others;
  } else {
    const float zt = target_z[row] * kLn2;
    if (zt == -kInf) {  // the target is left out
      loss[row] = sum == sum ? kInf : sum;
      lse[row] = others;
    } else {
      const float a = others - zt;
      const float tail = log1pf(expf(-fabsf(a)));
      loss[row] = fmaxf(a, 0.0f) + tail + (a != a ? a : 0.0f);
      lse[row] = fmaxf(others, zt) + tail;
    }
  }
}

// One block: the reduced loss and its divisor, summed in 64 bits in a fixed
// order.
__global__ void __launch_bounds__(1024) xent_total_kernel(const float* __restrict__ loss,
                                                          const int64_t* __restrict__ targets, int64_t ignore_index,
                                                          int64_t t, int mean, float* __restrict__ total,
                                                          float* __restrict__ divisor_out) {
  __shared__ double s_sum[32];
  __shared__ long long s_count[32];
  double sum = 0.0;
  long long count = 0;
  for (int64_t i = threadIdx.x; i < t; i += 1024)
    if (targets[i] != ignore_index) {
      sum += loss[i];
      ++count;
    }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, s);
    count += __shfl_xor_sync(0xffffffffu, count, s);
  }
  if ((threadIdx.x & 31) == 0) {
    s_sum[threadIdx.x >> 5] = sum;
    s_count[threadIdx.x >> 5] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) {
      sum += s_sum[w];
      count += s_count[w];
    }
    const double divisor = mean ? static_cast<double>(count) : 1.0;
    total[0] = static_cast<float>(sum / divisor);
    divisor_out[0] = static_cast<float>(divisor);
  }
}

// One block: the queries' factors relative to the largest gradient, and what
// the products are multiplied by at the end.
__global__ void __launch_bounds__(1024) xent_factors_kernel(const float* __restrict__ loss,
                                                            const float* __restrict__ lse,
                                                            const float* __restrict__ grad, int grad_stride,
                                                            const float* __restrict__ divisor,
                                                            const int64_t* __restrict__ targets, int64_t ignore_index,
                                                            int64_t t, int64_t v, float scale, float lift,
                                                            float* __restrict__ lse2, float* __restrict__ row_factor,
                                                            float* __restrict__ target_g,
                                                            float* __restrict__ out_scale) {
  __shared__ float s_top[32];
  float top = 0.0f;
  if (grad_stride == 0) {
    top = fabsf(grad[0]);
  } else {
    for (int64_t i = threadIdx.x; i < t; i += 1024)
      if (targets[i] != ignore_index) top = fmaxf(top, fabsf(grad[i]));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 32; ++w) top = fmaxf(top, s_top[w]);
  }
  if (threadIdx.x == 0) out_scale[0] = top * scale / lift / (divisor != nullptr ? divisor[0] : 1.0f);
  for (int64_t i = threadIdx.x; i < t; i += 1024) {
    const int64_t y = targets[i];
    const float g = grad[grad_stride == 0 ? 0 : i];
    const bool used = y != ignore_index && y >= 0 && y < v;
    row_factor[i] = used && top != 0.0f ? g / top * lift : 0.0f;
    // exp(-loss) - 1 is the target's share minus one, without cancellation.
    target_g[i] = expm1f(-loss[i]);
    lse2[i] = lse[i] == -kInf ? kInf : lse[i] * kLog2e;
  }
}

// The sum of dq's slabs, scaled and rounded to the queries' type.
template <bool BF>
__global__ void __launch_bounds__(256) xent_grad_q_kernel(const float* __restrict__ slab, int splits, int64_t slab_rows,
                                                          int64_t ld_slab, int64_t t, int d,
                                                          const float* __restrict__ out_scale, uint16_t* __restrict__ out,
                                                          int64_t ldo) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int quads = (d + 3) / 4;
  if (i >= t * quads) return;
  const int64_t row = i / quads;
  const int col = static_cast<int>(i - row * quads) * 4;
  const float4* s = reinterpret_cast<const float4*>(slab + row * ld_slab + col);
  const int64_t step = slab_rows * ld_slab / 4;
  float4 sum = s[0];
#pragma unroll 4
  for (int k = 1; k < splits; ++k) {
    const float4 w = s[k * step];
    sum.x += w.x;
    sum.y += w.y;
    sum.z += w.z;
    sum.w += w.w;
  }
  const float f = out_scale[0];
  const uint32_t lo = pack2<BF>(sum.x * f, sum.y * f), hi = pack2<BF>(sum.z * f, sum.w * f);
  uint16_t* o = out + row * ldo + col;
  if (col + 4 <= d && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
    *reinterpret_cast<uint2*>(o) = make_uint2(lo, hi);
  } else {
    o[0] = static_cast<uint16_t>(lo);
    if (col + 1 < d) o[1] = static_cast<uint16_t>(lo >> 16);
    if (col + 2 < d) o[2] = static_cast<uint16_t>(hi);
    if (col + 3 < d) o[3] = static_cast<uint16_t>(hi >> 16);
  }
}

template <int ROLE>
cudaError_t launch_role(const CUtensorMap* maps, const Args& p, bool bf, int clusters, cudaStream_t stream) {
  const bool bias = (ROLE == kStats || ROLE == kWeights) && p.bias != nullptr;
  constexpr bool kB = ROLE == kStats || ROLE == kWeights;
  auto kern = bf ? (bias ? xent_gemm_kernel<ROLE, true, kB> : xent_gemm_kernel<ROLE, true, false>)
                 : (bias ? xent_gemm_kernel<ROLE, false, kB> : xent_gemm_kernel<ROLE, false, false>);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
  if (e != cudaSuccess) return e;
  const int n = p.n_items < clusters ? p.n_items : clusters;
  kern<<<2 * n, kThreads, kSmem, stream>>>(maps[0], maps[1], p);
  return cudaGetLastError();
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Splits of the base for the forward: those whose items (query tile, split)
// take the fewest base tiles of the busiest pair, an item's start and end
// counted as one more tile.
int stats_splits(int64_t m_tiles, int64_t n_tiles, int clusters) {
  int best = 1;
  int64_t best_cost = 0;
  for (int s = 1; s <= 4 * clusters && s <= n_tiles; ++s) {
    const int64_t per = ceil_div(n_tiles, s);
    if (ceil_div(n_tiles, per) != s) continue;
    const int64_t cost = ceil_div(m_tiles * s, clusters) * (per + 1);
    if (best_cost == 0 || cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

// Columns of the base per piece of the backward: a G of 64 MB at most, whole
// tiles, at least four of them.
constexpr int64_t kPieceBytes = int64_t(64) << 20;
int64_t piece_cols(int64_t t, int64_t v) {
  const int64_t fit = kPieceBytes / 2 / t / kTile * kTile;
  const int64_t cols = fit < 4 * kTile ? 4 * kTile : fit;
  const int64_t all = align_up(v, kTile);
  if (all <= cols) return all;
  // Equal pieces: the last one is not left with a sliver.
  return align_up(ceil_div(all, ceil_div(all, cols)), kTile);
}

// Tiles of the gradients' N side (d columns): equal widths, a multiple of 32.
struct GradTiles {
  int n_tiles, n_cols;
  explicit GradTiles(int d) {
    n_tiles = static_cast<int>(ceil_div(d, kTile));
    n_cols = static_cast<int>(align_up(ceil_div(d, n_tiles), 32));
  }
};

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

struct ForwardWs {
  float2* part;
  float* target_z;
  int64_t bytes;
  ForwardWs(char* base, int64_t t, int splits) {
    Carve c{base};
    part = c.take<float2>(t * splits * 2);
    target_z = c.take<float>(t);
    bytes = c.used;
  }
};

struct BackwardWs {
  float *lse2, *row_factor, *target_g, *out_scale, *slab;
  uint16_t* g;
  int64_t bytes;
  BackwardWs(char* base, int64_t t, int64_t piece, int splits, int64_t slab_rows, int64_t ld_slab) {
    Carve c{base};
    lse2 = c.take<float>(t);
    row_factor = c.take<float>(t);
    target_g = c.take<float>(t);
    out_scale = c.take<float>(1);
    slab = c.take<float>(splits * slab_rows * ld_slab);
    g = c.take<uint16_t>(t * piece);
    bytes = c.used;
  }
};

}  // namespace

int64_t xent_forward_workspace(int64_t t, int64_t v, int clusters) {
  return ForwardWs(nullptr, t, stats_splits(ceil_div(t, kTile), ceil_div(v, kTile), clusters)).bytes;
}

int64_t xent_backward_workspace(int64_t t, int64_t v, int d, int clusters) {
  const GradTiles gt(d);
  const int64_t piece = piece_cols(t, v), m_tiles = ceil_div(t, kTile);
  return BackwardWs(nullptr, t, piece, grad_q_splits(m_tiles, gt.n_tiles, piece / kSlice, clusters), m_tiles * kTile,
                    static_cast<int64_t>(gt.n_tiles) * gt.n_cols)
      .bytes;
}

cudaError_t launch_xent_forward(const XentProblem& x, float* loss, float* lse, int reduction, float* total,
                                float* divisor, void* ws, int clusters, cudaStream_t stream, int* launches) {
  Args p = {};
  p.t = x.t;
  p.v = x.v;
  p.d = x.d;
  p.m_tiles = static_cast<int>(ceil_div(x.t, kTile));
  p.n_tiles = static_cast<int>(ceil_div(x.v, kTile));
  p.splits = stats_splits(p.m_tiles, p.n_tiles, clusters);
  p.per_split = static_cast<int>(ceil_div(p.n_tiles, p.splits));
  p.n_items = p.m_tiles * p.splits;
  p.n_cols = kTile;
  p.k_slices = static_cast<int>(ceil_div(x.d, kSlice));
  const bool bf = x.type == kElemBf16;
  p.idesc = tc::idesc_16(bf, false, false, kTile, kTile);
  p.c = x.scale * kLog2e;
  p.bias = x.bias;
  p.targets = x.targets;
  p.ignore_index = x.ignore_index;
  const ForwardWs w(static_cast<char*>(ws), x.t, p.splits);
  p.part = w.part;
  p.target_z = w.target_z;
  CUtensorMap maps[2];
  cudaError_t e = encode_rows_map(&maps[0], x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kHalf);
  if (e == cudaSuccess) e = encode_rows_map(&maps[1], x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kHalf);
  if (e == cudaSuccess) e = launch_role<kStats>(maps, p, bf, clusters, stream);
  if (e != cudaSuccess) return e;
  xent_join_kernel<<<static_cast<unsigned>(ceil_div(x.t, 8)), 256, 0, stream>>>(
      w.part, 2 * p.splits, w.target_z, x.targets, x.ignore_index, x.t, x.v, loss, lse);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  *launches = 2;
  if (reduction != 0) {
    xent_total_kernel<<<1, 1024, 0, stream>>>(loss, x.targets, x.ignore_index, x.t, reduction == 2, total, divisor);
    e = cudaGetLastError();
    *launches = 3;
  }
  return e;
}

cudaError_t launch_xent_backward(const XentProblem& x, const float* loss, const float* lse, const float* grad,
                                 int grad_stride, const float* divisor, void* dq, int64_t lddq, void* drows,
                                 int64_t lddr, void* ws, int clusters, cudaStream_t stream, int* launches) {
  const bool bf = x.type == kElemBf16;
  const GradTiles gt(x.d);
  const int64_t piece_max = piece_cols(x.t, x.v);
  const int m_tiles = static_cast<int>(ceil_div(x.t, kTile));
  const int64_t slab_rows = static_cast<int64_t>(m_tiles) * kTile;
  const int64_t ld_slab = static_cast<int64_t>(gt.n_tiles) * gt.n_cols;
  const int q_splits = grad_q_splits(m_tiles, gt.n_tiles, piece_max / kSlice, clusters);
  const BackwardWs w(static_cast<char*>(ws), x.t, piece_max, q_splits, slab_rows, ld_slab);
  xent_factors_kernel<<<1, 1024, 0, stream>>>(loss, lse, grad, grad_stride, divisor, x.targets, x.ignore_index, x.t, x.v,
                                              x.scale, bf ? 1.0f : 16384.0f, w.lse2, w.row_factor, w.target_g,
                                              w.out_scale);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  *launches = 1;

  Args base = {};
  base.t = x.t;
  base.v = x.v;
  base.d = x.d;
  base.targets = x.targets;
  base.ignore_index = x.ignore_index;
  base.c = x.scale * kLog2e;
  base.bias = x.bias;
  base.lse2 = w.lse2;
  base.row_factor = w.row_factor;
  base.target_g = w.target_g;
  base.g = w.g;
  base.ldg = piece_max;
  base.out_scale = w.out_scale;

  CUtensorMap weights[2];
  e = encode_rows_map(&weights[0], x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kHalf);
  if (e == cudaSuccess) e = encode_rows_map(&weights[1], x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kHalf);
  // MN-major operands: boxes of 64 columns by 64 rows.
  CUtensorMap rows_mn, q_mn;
  if (e == cudaSuccess) e = encode_rows_map(&rows_mn, x.type, x.rows, x.d, x.v, x.ldr * 2, kSlice, kSlice);
  if (e == cudaSuccess) e = encode_rows_map(&q_mn, x.type, x.q, x.d, x.t, x.ldq * 2, kSlice, kSlice);
  if (e != cudaSuccess) return e;
  int splits_used = 0;
  for (int64_t v0 = 0; v0 < x.v; v0 += piece_max) {
    const int64_t piece = x.v - v0 < piece_max ? x.v - v0 : piece_max;
    base.v0 = v0;
    base.piece = piece;
    // G of this piece.
    Args p = base;
    p.m_tiles = m_tiles;
    p.n_tiles = static_cast<int>(ceil_div(piece, kTile));
    p.n_items = p.m_tiles * p.n_tiles;
    p.n_cols = kTile;
    p.k_slices = static_cast<int>(ceil_div(x.d, kSlice));
    p.idesc = tc::idesc_16(bf, false, false, kTile, kTile);
    e = launch_role<kWeights>(weights, p, bf, clusters, stream);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (dq != nullptr) {
      p = base;
      p.m_tiles = m_tiles;
      p.n_tiles = gt.n_tiles;
      p.n_cols = gt.n_cols;
      p.k_slices = static_cast<int>(ceil_div(piece, kSlice));
      p.per_split = static_cast<int>(ceil_div(p.k_slices, q_splits));
      p.splits = static_cast<int>(ceil_div(p.k_slices, p.per_split));
      if (splits_used == 0) splits_used = p.splits;
      p.n_items = p.m_tiles * p.n_tiles * p.splits;
      p.idesc = tc::idesc_16(bf, false, true, kTile, gt.n_cols);
      p.slab = w.slab;
      p.ld_slab = ld_slab;
      p.accumulate = v0 > 0;
      CUtensorMap maps[2];
      e = encode_rows_map(&maps[0], x.type, w.g, piece, x.t, piece_max * 2, kSlice, kHalf);
      maps[1] = rows_mn;
      if (e == cudaSuccess) e = launch_role<kGradQ>(maps, p, bf, clusters, stream);
      if (e != cudaSuccess) return e;
      ++*launches;
    }
    if (drows != nullptr) {
      p = base;
      p.m_tiles = static_cast<int>(ceil_div(piece, kTile));
      p.n_tiles = gt.n_tiles;
      p.n_cols = gt.n_cols;
      p.k_slices = static_cast<int>(ceil_div(x.t, kSlice));
      p.n_items = p.m_tiles * p.n_tiles;
      p.idesc = tc::idesc_16(bf, true, true, kTile, gt.n_cols);
      p.out = drows;
      p.ldo = lddr;
      p.vec_out = reinterpret_cast<uintptr_t>(drows) % 16 == 0 && lddr % 8 == 0;
      CUtensorMap maps[2];
      e = encode_rows_map(&maps[0], x.type, w.g, piece, x.t, piece_max * 2, kSlice, kSlice);
      maps[1] = q_mn;
      if (e == cudaSuccess) e = launch_role<kGradRows>(maps, p, bf, clusters, stream);
      if (e != cudaSuccess) return e;
      ++*launches;
    }
  }
  if (dq != nullptr) {
    const int64_t work = x.t * ceil_div(x.d, 4);
    auto kern = bf ? xent_grad_q_kernel<true> : xent_grad_q_kernel<false>;
    kern<<<static_cast<unsigned>(ceil_div(work, 256)), 256, 0, stream>>>(w.slab, splits_used, slab_rows, ld_slab, x.t, x.d,
                                                                         w.out_scale, static_cast<uint16_t*>(dq), lddq);
    e = cudaGetLastError();
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
