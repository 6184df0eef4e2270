// Scores of 8-bit rows: the whole matrix
//     out[i][j] = (sum_l q[i][l] * x[j][l]) * q_scale[i] * x_scale[j] + bias[j]
// of m queries and n base rows, the sums exact in 32-bit integers
// (tcgen05.mma kind::i8), the scales and the bias applied in fp32 in the
// epilogue, one rounding to the output's type.
//
// Layout. A cluster of two CTAs computes 256 base rows x N queries per tile
// (N <= 256) with cta_group::2: base rows are the M side, one TMEM lane each,
// so the 32 lanes of an epilogue warp hold 32 neighbouring base rows of one
// query and every store is a run of a row of `out` straight from registers,
// with no transposition through shared memory. Each CTA stages its 128 base
// rows and half of the queries in slices of 128 codes (128-byte swizzle).
//
// What bounds it: the matrix itself. At 4 bytes a score the write takes longer
// than the products for d up to about 1000, with few queries the base's read
// is what remains. So the queries are kept in shared memory across base tiles
// where they fit (KC slices of N/2 rows; d <= 896 at N = 256), and only base
// rows stream through the ring.
//
// Tiles are numbered query group major and dealt to the clusters in equal
// contiguous runs, so a cluster changes its resident queries at most once more
// than it must, and the clusters of different query groups read the same base
// rows from L2.
//
// CTA roles (576 threads): warp 0 TMA producer, warp 1 TMEM owner and (even
// CTA) MMA issuer, warps 2-17 epilogue: four per TMEM quarter, on alternate
// blocks of 32 queries. Two accumulators (512 TMEM
// columns) overlap the epilogue with the next tile. Barriers as in the bf16
// candidate pass (k_gemm.cu); every wait is bounded, and a wait that gives up
// makes the tiles it concerns NaN and raises the operators' error word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "px_rows.cuh"
#include "px_rows.h"

namespace px {

namespace {

// Set when a bounded wait gave up (px_rows_status_device reads and clears it).
__device__ unsigned g_int8_err;

constexpr int kRows = 128;        // base rows per CTA and tile
constexpr int kSlice = 128;       // codes per slice
constexpr int kA = kRows * kSlice;  // 16 KB
constexpr int kMaxStages = 12;
constexpr int kGroups = 4;        // epilogue warps per TMEM quarter
constexpr int kEpiWarps = 4 * kGroups;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kWarpScales = 256 / kGroups;  // query scales an epilogue warp needs
constexpr int kMaxAccs = 8;
constexpr int kBars = 2 * kMaxStages + 2 * kMaxAccs + 4;  // one spare: the scales after them stay 16-byte aligned
constexpr size_t kFixed = 1024 + kBars * 8 + 16 + kEpiWarps * kWarpScales * 4;
constexpr size_t kSmemLimit = 232448;  // 227 KB

struct Params {
  const float* q_scale;
  const float* x_scale;
  const float* bias;
  void* out;
  int64_t ldo, m, n;
  int tiles;       // query groups x base tiles
  int base_tiles;
  int n_cols;      // queries per tile: a multiple of 32, at most 256
  int kc;          // slices
  int resident;    // queries stay in shared memory
  int stages, stage_bytes;
  int accs;        // accumulators, 512 / accs columns each
};

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The scores of queries j and j + 1 and this lane's base row.
__device__ __forceinline__ F2 two_scores(const uint32_t (&v)[32], int j, float w0, float w1, F2 xs, F2 bias) {
  return fma2(f2(static_cast<float>(static_cast<int>(v[j])), static_cast<float>(static_cast<int>(v[j + 1]))),
              mul2(f2(w0, w1), xs), bias);
}

// A pair's word of 16-bit scores: the even lane's both rows of query j, the
// odd lane's of query j + 1.
template <typename OT>
__device__ __forceinline__ uint32_t trade(float s0, float s1, int odd) {
  const uint32_t mine = pack2<OT>(s0, s1);
  const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
  return __byte_perm(mine, other, odd ? 0x3276 : 0x5410);
}

// Stores a block's scores, all 32 base rows of the warp being real. SOME: only
// the first `count` queries are. The stores evict first: the matrix is larger
// than what L2 should keep for the base.
template <typename OT, bool PAIR, int SOME>
__device__ __forceinline__ void store_queries(const uint32_t (&v)[32], const float* qs, float xs, float bias, OT* o,
                                              int64_t ldo, int odd, int count) {
  const float4* qs4 = reinterpret_cast<const float4*>(qs);
  const F2 xs2 = f2(xs, xs), bias2 = f2(bias, bias);
#pragma unroll
  for (int j4 = 0; j4 < 8; ++j4) {
    if (SOME && 4 * j4 >= count) break;
    const float4 w = qs4[j4];
    float s[4];
    unpack(two_scores(v, 4 * j4, w.x, w.y, xs2, bias2), s[0], s[1]);
    unpack(two_scores(v, 4 * j4 + 2, w.z, w.w, xs2, bias2), s[2], s[3]);
    if constexpr (PAIR) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t word = trade<OT>(s[2 * h], s[2 * h + 1], odd);
        if (!SOME || 4 * j4 + 2 * h + odd < count) __stcs(reinterpret_cast<uint32_t*>(o), word);
        o += 2 * ldo;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (!SOME || 4 * j4 + h < count) __stcs(o, narrow<OT>(s[h]));
        o += ldo;
      }
    }
  }
}

// The same for the base's last rows.
template <typename OT, bool PAIR>
__device__ __forceinline__ void store_ragged(const uint32_t (&v)[32], const float* qs, float xs, float bias, OT* o,
                                             int64_t ldo, int odd, int count, int keep) {
  const F2 xs2 = f2(xs, xs), bias2 = f2(bias, bias);
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    if (j >= count) break;
    float s0, s1;
    unpack(two_scores(v, j, qs[j], qs[j + 1], xs2, bias2), s0, s1);
    if constexpr (PAIR) {
      const uint32_t word = trade<OT>(s0, s1, odd);
      if (j + odd < count && keep == 2) *reinterpret_cast<uint32_t*>(o) = word;
      if (j + odd < count && keep == 1) *reinterpret_cast<unsigned short*>(o) = static_cast<unsigned short>(word);
    } else {
      if (keep > 0) *o = narrow<OT>(s0);
      if (keep > 0 && j + 1 < count) o[ldo] = narrow<OT>(s1);
    }
    o += 2 * ldo;
  }
}

// PAIR: 16-bit scores leave in pairs of base rows (out and its rows 4-byte
// aligned).
template <typename OT, bool PAIR>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
int8_scores_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_q,
                   const Params p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int b_slice = p.n_cols / 2 * kSlice;  // bytes of a slice of this CTA's queries
  const int b_bytes = p.resident ? p.kc * b_slice : 0;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + b_bytes + p.stages * p.stage_bytes);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  float* s_scale = reinterpret_cast<float*>(s_tmem + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t smem_base = tc::smem_addr(smem);
  const uint32_t ring = smem_base + b_bytes;
  auto full_bar = [&](int s) { return tc::smem_addr(&bars[s]); };
  auto empty_bar = [&](int s) { return tc::smem_addr(&bars[kMaxStages + s]); };
  auto tfull_bar = [&](int a) { return tc::smem_addr(&bars[2 * kMaxStages + a]); };
  auto tempty_bar = [&](int a) { return tc::smem_addr(&bars[2 * kMaxStages + kMaxAccs + a]); };
  const uint32_t bfull_bar = tc::smem_addr(&bars[2 * kMaxStages + 2 * kMaxAccs]);       // resident queries loaded
  const uint32_t bempty_bar = tc::smem_addr(&bars[2 * kMaxStages + 2 * kMaxAccs + 1]);  // and no longer read
  const uint32_t done_bar = tc::smem_addr(&bars[2 * kMaxStages + 2 * kMaxAccs + 2]);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < p.accs; ++a) {
      tc::mbar_init(tfull_bar(a), 1);
      tc::mbar_init(tempty_bar(a), 2 * kEpiWarps);
    }
    tc::mbar_init(bfull_bar, 1);
    tc::mbar_init(bempty_bar, 1);
    tc::mbar_init(done_bar, 1);
    *s_abort = 0;
    tc::fence_mbarrier_init_cluster();
  }
  if (warp == 0 && lane == 0) {
    tc::prefetch_tmap(&tm_x);
    tc::prefetch_tmap(&tm_q);
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
  const int acc_cols = 512 / p.accs;
  wait_for_previous();
  let_next_start();
  const int64_t cluster = tc::cluster_id_x();
  const int64_t nclusters = tc::nclusters_x();
  const int t0 = static_cast<int>(p.tiles * cluster / nclusters);
  const int t1 = static_cast<int>(p.tiles * (cluster + 1) / nclusters);
  // Query group and base tile of t0; the roles count on from there.
  const int group0 = t0 / p.base_tiles;
  const int base0 = t0 - group0 * p.base_tiles;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int64_t loads = 0;  // ring slots filled so far: load l uses stage l % stages
      int stage = 0;
      uint32_t phase = 0;
      bool fresh = true;    // the queries changed
      uint32_t groups = 0;  // resident query groups loaded so far
      int qg = group0, bt = base0;
      bool ok = true;
      for (int t = t0; ok && t < t1; ++t) {
        const int q0 = qg * p.n_cols + static_cast<int>(rank) * (p.n_cols / 2);
        const int r0 = bt * (2 * kRows) + static_cast<int>(rank) * kRows;
        if (p.resident && fresh) {
          if (groups > 0 && !tc::mbar_wait(bempty_bar, (groups - 1) & 1, s_abort)) break;
          const uint32_t fb = tc::mapa_shared(bfull_bar, 0);
          if (leader) tc::mbar_arrive_expect_tx(bfull_bar, 2 * b_bytes);
          for (int kc = 0; kc < p.kc; ++kc)
            tc::tma_load_2d_pair(smem_base + kc * b_slice, &tm_q, fb, kc * kSlice, q0);
          fresh = false;
          ++groups;
        }
        for (int kc = 0; kc < p.kc; ++kc) {
          if (!tc::mbar_wait(empty_bar(stage), phase ^ 1, s_abort)) {
            ok = false;
            break;
          }
          const uint32_t dst = ring + stage * p.stage_bytes;
          const uint32_t fb = tc::mapa_shared(full_bar(stage), 0);
          if (leader) tc::mbar_arrive_expect_tx(full_bar(stage), 2 * p.stage_bytes);
          tc::tma_load_2d_pair(dst, &tm_x, fb, kc * kSlice, r0);
          if (!p.resident) tc::tma_load_2d_pair(dst + kA, &tm_q, fb, kc * kSlice, q0);
          ++loads;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (++bt == p.base_tiles) {
          bt = 0;
          ++qg;
          fresh = true;
        }
      }
      // Both CTAs' loads complete on the even CTA's barriers: it waits for
      // the last phase of each before shared memory goes away.
      if (leader) {
        for (int64_t l = loads > p.stages ? loads - p.stages : 0; l < loads; ++l)
          quiet_wait(full_bar(static_cast<int>(l % p.stages)), static_cast<uint32_t>(l / p.stages) & 1);
        if (groups > 0) quiet_wait(bfull_bar, (groups - 1) & 1);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (even CTA)
    // The whole warp walks the loop, so that descriptors and addresses stay in
    // uniform registers (issued by a lone lane, a slice's four MMAs took about
    // 900 clocks of address arithmetic); one elected lane issues.
    if (leader) {
      const bool issuer = tc::elect_one();
      const uint32_t idesc = tc::idesc_s8(2 * kRows, p.n_cols);
      const uint64_t kind = tc::sw128_kmajor_desc(0);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool fresh = true;
      uint32_t groups = 0;
      int bt = base0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, s_abort)) != 0;
      };
      for (int t = t0; ok && t < t1; ++t) {
        if (!wait(tempty_bar(acc), acc_phase ^ 1)) break;
        if (p.resident && fresh) {
          if (!wait(bfull_bar, groups & 1)) break;
          fresh = false;
          ++groups;
        }
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * acc_cols);
        for (int kc = 0; kc < p.kc; ++kc) {
          if (!wait(full_bar(stage), phase)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t a_addr = ring + stage * p.stage_bytes;
          const uint64_t a_desc = kind + (a_addr >> 4);
          const uint64_t b_desc = kind + ((p.resident ? smem_base + kc * b_slice : a_addr + kA) >> 4);
          if (issuer) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_s8_pair(d_tmem, a_desc + 2 * kk, b_desc + 2 * kk, idesc, (kc > 0 || kk > 0) ? 1u : 0u);
            tc::mma_commit_pair_both(empty_bar(stage));
          }
          __syncwarp();
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (issuer) tc::mma_commit_pair_both(tfull_bar(acc));
        if (++bt == p.base_tiles) {
          bt = 0;
          fresh = true;
          if (issuer && p.resident && t + 1 < t1) tc::mma_commit_pair_both(bempty_bar);
        }
        __syncwarp();
        if (++acc == p.accs) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (issuer) tc::mma_commit_pair_both(done_bar);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int grp = (warp - 2) >> 2;  // which blocks of 32 queries: grp, grp + 4
    const int quarter = warp & 3;     // TMEM lanes this warp may access
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    float* scale = s_scale + (warp - 2) * kWarpScales;
    OT* out = static_cast<OT*>(p.out);
    int acc = 0;
    uint32_t acc_phase = 0;
    int qg = group0, bt = base0;
    bool fresh = true;  // the queries changed
    bool lost = false;  // a wait gave up: the scores that remain are NaN
    float next_xs, next_bias;
    auto load_row = [&](int tile) {
      const int64_t r = static_cast<int64_t>(tile) * (2 * kRows) + rank * kRows + quarter * 32 + lane;
      next_xs = r < p.n ? __ldg(p.x_scale + r) : 0.0f;
      next_bias = r < p.n && p.bias != nullptr ? __ldg(p.bias + r) : 0.0f;
    };
    load_row(bt);
    for (int t = t0; t < t1; ++t) {
      const int64_t q0 = static_cast<int64_t>(qg) * p.n_cols;
      const int64_t row = static_cast<int64_t>(bt) * (2 * kRows) + rank * kRows + quarter * 32 + lane;
      if (fresh) {
        __syncwarp();
#pragma unroll
        for (int b = 0; b < kWarpScales / 32; ++b) {
          const int64_t qi = q0 + (kGroups * b + grp) * 32 + lane;
          scale[b * 32 + lane] = qi < p.m ? __ldg(p.q_scale + qi) : 0.0f;
        }
        __syncwarp();
        fresh = false;
      }
      float xs = next_xs;
      const float bias = next_bias;
      // The next tile's, one tile ahead of its use.
      load_row(bt + 1 == p.base_tiles ? 0 : bt + 1);
      if (!lost && !__all_sync(0xffffffffu, tc::mbar_wait(tfull_bar(acc), acc_phase, s_abort))) lost = true;
      if (lost) xs = __int_as_float(0x7fc00000);
      tc::tc_fence_after();
      const int64_t row_warp = row - lane;
      // This warp's blocks: grp, grp + 4 of the tile's that hold queries.
      const int queries = p.m - q0 < p.n_cols ? static_cast<int>(p.m - q0) : p.n_cols;
      const int blocks = row_warp < p.n ? (queries + 31) / 32 : 0;
      for (int b = grp; b < blocks; b += kGroups) {
        __syncwarp();
        uint32_t v[32];
        tc::tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * acc_cols + b * 32), v);
        tc::tmem_ld_wait();
        if (b + kGroups >= blocks) {
          // The warp's last columns are in registers: the accumulator is free.
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
        }
        const int64_t qb = q0 + b * 32;
        const float* qs = scale + b / kGroups * 32;
        const int count = queries - b * 32 < 32 ? queries - b * 32 : 32;
        // Lanes 2i and 2i + 1 trade 16-bit scores when these leave in pairs:
        // the even one stores both rows' of query j, the odd one of j + 1.
        const int odd = PAIR ? lane & 1 : 0;
        OT* o = out + (qb + odd) * p.ldo + (row - odd);
        if (row_warp + 32 <= p.n) {
          if (count == 32) {
            store_queries<OT, PAIR, 0>(v, qs, xs, bias, o, p.ldo, odd, 32);
          } else {
            store_queries<OT, PAIR, 1>(v, qs, xs, bias, o, p.ldo, odd, count);
          }
        } else {
          // The last base rows. keep: this lane's pair exists (2), or its
          // first row alone (1: the last of an odd count), or nothing (0).
          const int64_t left = p.n - (row - odd);
          store_ragged<OT, PAIR>(v, qs, xs, bias, o, p.ldo, odd, count,
                                 left >= 2 ? 2 : left < 0 ? 0 : static_cast<int>(left));
        }
      }
      if (grp >= blocks) {  // nothing to read in this tile
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
      }
      if (++acc == p.accs) {
        acc = 0;
        acc_phase ^= 1;
      }
      if (++bt == p.base_tiles) {
        bt = 0;
        ++qg;
        fresh = true;
      }
    }
  }

  if (warp == 1 && lane == 0) quiet_wait(done_bar, 0);
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 512);
  if (threadIdx.x == 0 && *s_abort) atomicOr(&g_int8_err, 1u);
}

template <typename OT, bool PAIR>
cudaError_t launch_typed(const CUtensorMap* maps, const Params& p, int clusters, size_t smem, cudaStream_t stream) {
  auto kern = int8_scores_kernel<OT, PAIR>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  return launch_after(kern, 2 * clusters, kThreads, smem, stream, maps[0], maps[1], p);
}

}  // namespace

cudaError_t launch_int8_scores(const Int8ScoresArgs& a, int clusters, cudaStream_t stream) {
  Params p;
  p.q_scale = a.q_scale;
  p.x_scale = a.x_scale;
  p.bias = a.bias;
  p.out = a.out;
  p.ldo = a.ldo;
  p.m = a.m;
  p.n = a.n;
  // Query groups of equal size, a multiple of 32 (the pair's smallest N).
  const int64_t groups = (a.m + 255) / 256;
  p.n_cols = static_cast<int>(((a.m + groups - 1) / groups + 31) / 32 * 32);
  p.base_tiles = static_cast<int>((a.n + 2 * kRows - 1) / (2 * kRows));
  // As many accumulators as fit: a tile of few queries is short, and what its
  // hand-overs take is hidden only by the tiles in flight.
  p.accs = p.n_cols <= 64 ? 8 : p.n_cols <= 128 ? 4 : 2;
  if (groups * p.base_tiles > 0x7fffffff) return cudaErrorInvalidValue;
  p.tiles = static_cast<int>(groups * p.base_tiles);
  p.kc = (a.d + kSlice - 1) / kSlice;
  const int b_slice = p.n_cols / 2 * kSlice;
  // Resident queries leave at least six ring stages, as many as the bf16
  // candidate pass has.
  p.resident = kFixed + static_cast<size_t>(p.kc) * b_slice + 6 * kA <= kSmemLimit;
  p.stage_bytes = p.resident ? kA : kA + b_slice;
  const size_t b_bytes = p.resident ? static_cast<size_t>(p.kc) * b_slice : 0;
  const int fit = static_cast<int>((kSmemLimit - kFixed - b_bytes) / p.stage_bytes);
  p.stages = fit < kMaxStages ? fit : kMaxStages;
  const size_t smem = kFixed + b_bytes + static_cast<size_t>(p.stages) * p.stage_bytes;
  CUtensorMap maps[2];
  cudaError_t e = encode_rows_map(&maps[0], kElemS8, a.x, a.d, a.n, a.ldx, kSlice, kRows, 128);
  if (e == cudaSuccess) e = encode_rows_map(&maps[1], kElemS8, a.q, a.d, a.m, a.ldq, kSlice, p.n_cols / 2, 128);
  if (e != cudaSuccess) return e;
  if (p.tiles < clusters) clusters = p.tiles;
  const bool pair = reinterpret_cast<uintptr_t>(a.out) % 4 == 0 && a.ldo % 2 == 0;
  switch (a.type) {
    case kElemF32: return launch_typed<float, false>(maps, p, clusters, smem, stream);
    case kElemF16:
      return pair ? launch_typed<__half, true>(maps, p, clusters, smem, stream)
                  : launch_typed<__half, false>(maps, p, clusters, smem, stream);
    case kElemBf16:
      return pair ? launch_typed<__nv_bfloat16, true>(maps, p, clusters, smem, stream)
                  : launch_typed<__nv_bfloat16, false>(maps, p, clusters, smem, stream);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t take_int8_error(cudaStream_t stream, unsigned* out) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(out, g_int8_err, sizeof(unsigned), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *out == 0) return e;
  const unsigned zero = 0;
  e = cudaMemcpyToSymbolAsync(g_int8_err, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, stream);
  return e == cudaSuccess ? cudaStreamSynchronize(stream) : e;
}

}  // namespace px
