// Scores of 8-bit rows: the whole matrix
//     out[i][j] = (sum_l q[i][l] * x[j][l]) * q_scale[i] * x_scale[j] + bias[j]
// of m queries and n base rows, the sums exact in 32-bit integers
// (tcgen05.mma kind::i8), the scales and the bias applied in fp32 in the
// epilogue, one rounding to the output's type.
//
// Layout. A cluster of two CTAs computes 256 base rows x N queries per tile
// (N <= 256) with cta_group::2: base rows are the M side, one TMEM lane each,
// so the 32 lanes of an epilogue warp hold 32 neighbouring base rows of one
// query, and four warps put a query's 128 of them side by side in shared memory
// without transposing: a run of 256 or 512 bytes of a row of `out`. Each CTA stages its 128 base
// rows and half of the queries in slices of 128 codes (128-byte swizzle).
//
// What bounds it: the matrix itself. At 4 bytes a score the write takes longer
// than the products for d up to about 1000, with few queries the base's read
// is what remains. So the queries are kept in shared memory across base tiles
// where they fit beside 80 KB of ring (KC slices of N/2 rows; at N = 256 d <= 768,
// or 1024 where nothing is staged), and only base rows stream through the ring.
// Measured, fp32 out: 64 x 1M x 128 in 75 us and 1000 x 100k x 384 in 97 us,
// 0.79 and 0.70 of what their bytes take at a copy's rate; longer runs per row
// of `out` (1 KB) did not change that. bf16 out: 10k x 100k x 768 in 804-818 us,
// 1.9 POP/s, under the power cap; 786 us back to back, 642 without its stores
// and 544 with no epilogue at all, and 677, 553 and 461 when the GPU is cool. So
// the epilogue and its stores take 216 us that the products do not hide.
//
// Order. Clusters form teams. The clusters of a team take neighbouring base
// tiles of one query group, so what is written at any time is long runs of 256
// rows of `out`: with a run of base tiles per cluster, whose writes lie far
// apart, plain stores of a 400 MB matrix reach 3.9 TB/s, with neighbouring
// tiles 5-6. The teams take different query groups at the same base tiles, so
// that they share what is read from HBM.
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
constexpr int kOutBuf = 8192;     // staging of an epilogue group's stores by TMA,
constexpr int kRaggedBuf = 8704;  // or of others: two halves of 8 fp32 or 16 16-bit rows and 16 bytes each
constexpr int kBlocks = 256 / 32 / kGroups;  // blocks of 32 columns per epilogue warp
constexpr int kWarpScales = 256 / kGroups;  // query scales an epilogue warp needs
constexpr int kMaxAccs = 8;
constexpr int kBars = 2 * kMaxStages + 2 * kMaxAccs + 4;  // one spare: the scales after them stay 16-byte aligned
constexpr size_t kFixed = 1024 + kBars * 8 + 16 + kEpiWarps * kWarpScales * 4;
constexpr size_t kSmemLimit = 232448;  // 227 KB
// From this size on, a matrix that TMA cannot address leaves through shared
// memory (us, from registers and staged): fp16 2705 x 49k (267 MB) 100 and 114,
// bf16 181 x 249k (90 MB) 48 and 53, fp32 129 x 425k (219 MB) 71 and 73; but
// fp16 210 x 969k (407 MB) 221 and 176, bf16 952 x 855k (1.6 GB) 878 and 612,
// fp32 1308 x 543k (2.8 GB) 1155 and 747.
constexpr int64_t kStagedBytes = int64_t(320) << 20;

struct Params {
  const float* q_scale;
  const float* x_scale;
  const float* bias;
  void* out;
  int64_t ldo, m, n;
  int groups;      // query groups
  int base_tiles;
  int teams, width;  // teams of `width` clusters; a team takes every teams-th query group
  int n_cols;      // queries per tile: a multiple of 32, at most 256
  int kc;          // slices
  int resident;    // queries stay in shared memory
  int subs;        // groups of 256 base rows per tile: subs * n_cols <= 256
  int stages, stage_bytes;
  int keep_base;   // base rows are read again: L2 should keep them
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
// The scores of queries j and j + 1 and this lane's base row. The sum is taken
// times the query's scale first: the scales' own product may leave the range of
// fp32 where the score does not.
__device__ __forceinline__ F2 two_scores(const uint32_t (&v)[32], int j, float w0, float w1, F2 xs, F2 bias) {
  return fma2(mul2(f2(static_cast<float>(static_cast<int>(v[j])), static_cast<float>(static_cast<int>(v[j + 1]))), f2(w0, w1)),
              xs, bias);
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

// Arrive and wait of one epilogue group's four warps.
__device__ __forceinline__ void group_sync(int grp) {
  asm volatile("bar.sync %0, 128;" ::"r"(grp + 1) : "memory");
}

// Stages a block's scores of the CTA's 128 base rows, with the group's other
// three warps, and stores them by TMA: rows of 128 scores, 16 queries of fp32
// or 32 of 16 bits at a time. Queries and base rows past the matrix are not
// written.
template <typename OT>
__device__ __forceinline__ void stage_queries(const uint32_t (&v)[32], const float* qs, float xs, float bias,
                                              uint32_t buf, int row_in_tile, int grp, int count,
                                              const CUtensorMap* map, int row_tile, int q) {
  const float4* qs4 = reinterpret_cast<const float4*>(qs);
  const F2 xs2 = f2(xs, xs), bias2 = f2(bias, bias);
  constexpr int kParts = sizeof(OT) / 2, kQueries = 32 / kParts;
  const uint32_t at = buf + row_in_tile * static_cast<int>(sizeof(OT));
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    if (part * kQueries >= count) break;
    if (row_in_tile == 0) store_wait_read();
    group_sync(grp);
#pragma unroll
    for (int i = 0; i < kQueries / 4; ++i) {
      const float4 w = qs4[part * (kQueries / 4) + i];
      const int j = part * kQueries + 4 * i;
      float s[4];
      unpack(two_scores(v, j, w.x, w.y, xs2, bias2), s[0], s[1]);
      unpack(two_scores(v, j + 2, w.z, w.w, xs2, bias2), s[2], s[3]);
      if constexpr (sizeof(OT) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + (4 * i + k) * (kRows * 4)), "f"(s[k]) : "memory");
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t both = pack2<OT>(s[2 * k], s[2 * k + 1]);
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + (4 * i + 2 * k) * (kRows * 2)),
                       "h"(static_cast<unsigned short>(both))
                       : "memory");
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + (4 * i + 2 * k + 1) * (kRows * 2)),
                       "h"(static_cast<unsigned short>(both >> 16))
                       : "memory");
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    group_sync(grp);
    if (row_in_tile == 0) {
      tma_store(map, buf, row_tile, q + part * kQueries);
      store_commit();
    }
  }
}

// The same for a large matrix that TMA cannot address (rows that begin or end
// off 16-byte boundaries): the warps store the rows of 128 scores themselves,
// in aligned 16-byte pieces and single scores at either end. A row lies in the
// buffer as far from a boundary as in `out`, so pieces are read whole. Stored
// straight from registers, 32 scores of a query per instruction, most of a
// row's sectors are written in two parts, which costs little while L2 joins
// them and much past it; kStagedBytes has the measurements. Tiles that overlap,
// so that a CTA stores whole sectors only, gained nothing.
// How far rows begin past a boundary repeats every kPiece queries, so that each
// thread works out once where its scores go and which pieces it stores.
template <typename OT>
struct Ragged {
  static constexpr int kSize = static_cast<int>(sizeof(OT)), kPiece = 16 / kSize;  // scores per piece
  static constexpr int kPitch = kRows * kSize + 16;
  static constexpr uint32_t kHalf = kRaggedBuf / 2;
  static constexpr int kQueries = kRaggedBuf / 2 / kPitch / 4 * 4;  // per half of the buffer
  static constexpr int kLanes = kRows / kPiece, kAtOnce = 32 / kLanes;  // lanes per row, rows per instruction
  static constexpr int kPerWarp = kQueries / 4 / kAtOnce;
  static_assert(kQueries % kPiece == 0 && (32 / kQueries) % 2 == 0, "parts");
  uint32_t place[kPiece];    // this thread's score of query j (modulo kPiece), in the buffer's first half
  uint32_t row[kPerWarp];    // where the rows this thread stores from begin there
  int piece[kPerWarp];       // the first score of its piece of a row
  int edge[kPerWarp];        // and the single one it stores of a whole row, or -1
  int in_part;               // its first row

  __device__ __forceinline__ Ragged(const OT* out, int64_t ldo, uint32_t buf, int row_in_tile) {
    const uint32_t step = static_cast<uint32_t>(ldo) * kSize;
    const uint32_t first = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(out));
    const int lane = row_in_tile & 31, l = lane % kLanes;
    in_part = (row_in_tile >> 5) * kPerWarp * kAtOnce + lane / kLanes;
#pragma unroll
    for (int j = 0; j < kPiece; ++j) place[j] = buf + row_in_tile * kSize + ((first + j * step) & 15);
#pragma unroll
    for (int i = 0; i < kPerWarp; ++i) {
      const int j = in_part + i * kAtOnce;
      const uint32_t past = (first + j * step) & 15;
      const int head = static_cast<int>((16 - past) & 15) / kSize;  // scores before the first boundary
      row[i] = buf + j * kPitch + past;
      piece[i] = head + l * kPiece;
      edge[i] = l < head ? l : l >= kPiece && l - kPiece < kPiece - head && head > 0 ? kRows - 2 * kPiece + head + l : -1;
    }
  }

  static __device__ __forceinline__ void single(OT* to, uint32_t from) {
    if constexpr (kSize == 4) {
      float x;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(from));
      *reinterpret_cast<float*>(to) = x;
    } else {
      unsigned short x;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x) : "r"(from));
      *reinterpret_cast<unsigned short*>(to) = x;
    }
  }

  // A block's scores: `count` queries of `rows` base rows, out the first's.
  __device__ __forceinline__ void store(const uint32_t (&v)[32], const float* qs, float xs, float bias, int grp,
                                        int count, OT* out, int64_t ldo, int rows) const {
    const float4* qs4 = reinterpret_cast<const float4*>(qs);
    const F2 xs2 = f2(xs, xs), bias2 = f2(bias, bias);
#pragma unroll
    for (int part = 0; part < 32 / kQueries; ++part) {
      if (part * kQueries >= count) {
        // The next block begins with the first half again, which the last part read.
        if (part & 1) group_sync(grp);
        break;
      }
#pragma unroll
      for (int i = 0; i < kQueries / 4; ++i) {
        const int j = part * kQueries + 4 * i;
        const float4 w = qs4[j / 4];
        float s[4];
        unpack(two_scores(v, j, w.x, w.y, xs2, bias2), s[0], s[1]);
        unpack(two_scores(v, j + 2, w.z, w.w, xs2, bias2), s[2], s[3]);
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const uint32_t at0 = place[(j + k) % kPiece], at1 = place[(j + k + 1) % kPiece];
          const uint32_t add = (part & 1) * kHalf + (4 * i + k) * kPitch;
          if constexpr (kSize == 4) {
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at0 + add), "f"(s[k]) : "memory");
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(at1 + add + kPitch), "f"(s[k + 1]) : "memory");
          } else {
            const uint32_t both = pack2<OT>(s[k], s[k + 1]);
            asm volatile("st.shared.b16 [%0], %1;" ::"r"(at0 + add), "h"(static_cast<unsigned short>(both)) : "memory");
            asm volatile("st.shared.b16 [%0], %1;" ::"r"(at1 + add + kPitch), "h"(static_cast<unsigned short>(both >> 16))
                         : "memory");
          }
        }
      }
      // Also: every warp has read what the other half held.
      group_sync(grp);
#pragma unroll
      for (int i = 0; i < kPerWarp; ++i) {
        const int j = part * kQueries + in_part + i * kAtOnce;
        if (j >= count) continue;
        OT* to = out + j * ldo;
        const uint32_t from = row[i] + (part & 1) * kHalf;
        if (piece[i] + kPiece <= rows) {
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                       : "r"(from + piece[i] * kSize));
          __stcs(reinterpret_cast<uint4*>(to + piece[i]), x);
        }
        if (rows == kRows) {
          if (edge[i] >= 0) single(to + edge[i], from + edge[i] * kSize);
        } else {
          // The base's last rows: those before the first boundary, and past the last whole piece.
          const int l = (threadIdx.x & 31) % kLanes, head = piece[i] - l * kPiece;
          if (l < min(head, rows)) single(to + l, from + l * kSize);
          if (piece[i] < rows && piece[i] + kPiece > rows)
            for (int e = piece[i]; e < rows; ++e) single(to + e, from + e * kSize);
        }
      }
    }
  }
};

// How scores leave: by TMA (rows of whole 16-byte pieces, on 16-byte
// boundaries), staged by the warps (large matrices of other rows), or straight
// from registers, 16-bit scores in pairs of base rows where out and its rows
// are 4-byte aligned.
enum Way { kTma, kStaged, kPairs, kSingle };
// Shared memory that an epilogue group stages in.
constexpr int staging(int way) { return way == kTma ? kOutBuf : way == kStaged ? kRaggedBuf : 0; }

template <typename OT, int WAY>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
int8_scores_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_q,
                   const __grid_constant__ CUtensorMap tm_out, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int b_slice = p.n_cols / 2 * kSlice;  // bytes of a slice of this CTA's queries
  const int b_bytes = p.resident ? p.kc * b_slice : 0;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + b_bytes + p.stages * p.stage_bytes + kGroups * staging(WAY));
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
  // This cluster's tiles: numbers first, first + width, ... of its team's.
  const int team = static_cast<int>(tc::cluster_id_x()) / p.width;
  const int first = static_cast<int>(tc::cluster_id_x()) % p.width;
  const int tiles = p.base_tiles * ((p.groups - team + p.teams - 1) / p.teams);
  const int base0 = first % p.base_tiles;
  const int group0 = team + first / p.base_tiles * p.teams;
  // The next tile: `width` base tiles on, in the team's next query group where
  // that passes the last; true if the queries changed.
  auto advance = [&](int& qg, int& bt) {
    bt += p.width;
    bool changed = false;
    while (bt >= p.base_tiles) {
      bt -= p.base_tiles;
      qg += p.teams;
      changed = true;
    }
    return changed;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int64_t loads = 0;  // ring slots filled so far: load l uses stage l % stages
      int stage = 0;
      uint32_t phase = 0;
      bool fresh = true;    // the queries changed
      const uint64_t policy = p.keep_base ? tc::l2_evict_last() : tc::l2_evict_first();
      uint32_t groups = 0;  // resident query groups loaded so far
      int qg = group0, bt = base0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += p.width) {
        const int q0 = qg * p.n_cols + static_cast<int>(rank) * (p.n_cols / 2);
        const int r0 = bt * p.subs * (2 * kRows) + static_cast<int>(rank) * kRows;
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
          for (int sub = 0; sub < p.subs; ++sub)
            tc::tma_load_2d_pair_hint(dst + sub * kA, &tm_x, fb, kc * kSlice, r0 + sub * (2 * kRows), policy);
          if (!p.resident) tc::tma_load_2d_pair(dst + p.subs * kA, &tm_q, fb, kc * kSlice, q0);
          ++loads;
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        fresh = advance(qg, bt) || fresh;
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
      int qg = group0, bt = base0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, s_abort)) != 0;
      };
      for (int t = first; ok && t < tiles; t += p.width) {
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
          const uint64_t b_desc = kind + ((p.resident ? smem_base + kc * b_slice : a_addr + p.subs * kA) >> 4);
          if (issuer) {
            for (int sub = 0; sub < p.subs; ++sub) {
              const uint64_t a_desc = kind + ((a_addr + sub * kA) >> 4);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                tc::mma_s8_pair(d_tmem + sub * p.n_cols, a_desc + 2 * kk, b_desc + 2 * kk, idesc,
                                (kc > 0 || kk > 0) ? 1u : 0u);
            }
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
        if (advance(qg, bt)) {
          fresh = true;
          if (issuer && p.resident && t + p.width < tiles) tc::mma_commit_pair_both(bempty_bar);
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
    const uint32_t out_buf = ring + p.stages * p.stage_bytes + grp * kOutBuf;
    const uint32_t ragged_buf = ring + p.stages * p.stage_bytes + grp * kRaggedBuf;
    const Ragged<OT> ragged(WAY == kStaged ? static_cast<const OT*>(p.out) : nullptr, p.ldo, ragged_buf,
                            quarter * 32 + lane);
    OT* out = static_cast<OT*>(p.out);
    int acc = 0;
    uint32_t acc_phase = 0;
    int qg = group0, bt = base0;
    bool fresh = true;  // the queries changed
    bool lost = false;  // a wait gave up: the scores that remain are NaN
    // This warp's blocks of 32 columns: grp and grp + 4 of the tile's, block b
    // being queries b % q_blocks of base rows b / q_blocks (divided here, once).
    const int q_blocks = p.n_cols / 32;
    const int row_in_cta = quarter * 32 + lane;
    int sub_of[kBlocks], q_of[kBlocks];  // row group and first query of each block
#pragma unroll
    for (int k = 0; k < kBlocks; ++k) {
      sub_of[k] = (grp + kGroups * k) / q_blocks;
      q_of[k] = (grp + kGroups * k - sub_of[k] * q_blocks) * 32;
    }
    float next_xs[kBlocks], next_bias[kBlocks];
    auto load_rows = [&](int tile) {
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int sub = sub_of[k];
        const int64_t r = (static_cast<int64_t>(tile) * p.subs + sub) * (2 * kRows) + rank * kRows + row_in_cta;
        const bool live = sub < p.subs && r < p.n;
        next_xs[k] = live ? p.x_scale[r] : 0.0f;
        next_bias[k] = live && p.bias != nullptr ? p.bias[r] : 0.0f;
      }
    };
    load_rows(bt);
    for (int t = first; t < tiles; t += p.width) {
      const int64_t q0 = static_cast<int64_t>(qg) * p.n_cols;
      // The next tile's base rows, whichever query group's it is.
      int wrapped = bt + p.width;
      while (wrapped >= p.base_tiles) wrapped -= p.base_tiles;
      if (fresh) {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
          const int64_t qi = q0 + q_of[k] + lane;
          scale[k * 32 + lane] = qi < p.m ? p.q_scale[qi] : 0.0f;
        }
        __syncwarp();
        fresh = false;
      }
      float xs[kBlocks], bias[kBlocks];
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        xs[k] = next_xs[k];
        bias[k] = next_bias[k];
      }
      // The next tile's, one tile ahead of their use.
      load_rows(wrapped);
      if (!lost && !__all_sync(0xffffffffu, tc::mbar_wait(tfull_bar(acc), acc_phase, s_abort))) lost = true;
      tc::tc_fence_after();
      const int queries = p.m - q0 < p.n_cols ? static_cast<int>(p.m - q0) : p.n_cols;
      bool freed = false;
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int b = grp + kGroups * k;
        const int sub = sub_of[k], q_in = q_of[k];
        const int64_t row_cta = (static_cast<int64_t>(bt) * p.subs + sub) * (2 * kRows) + rank * kRows;
        const int64_t row = row_cta + row_in_cta, row_warp = row - lane;
        // Where scores are staged, all four warps of a group take part, base rows
        // or not: they meet at barriers, and what lies past the matrix is left out.
        if (sub >= p.subs || q_in >= queries || (WAY <= kStaged ? row_cta >= p.n : row_warp >= p.n)) continue;  // warp-uniform
        __syncwarp();
        uint32_t v[32];
        tc::tmem_ld_32x32b_x32(lane_addr + static_cast<uint32_t>(acc * acc_cols + b * 32), v);
        tc::tmem_ld_wait();
        if (k == kBlocks - 1) {
          // The warp's last columns are in registers: the accumulator is free.
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
          freed = true;
        }
        const float row_scale = lost ? __int_as_float(0x7fc00000) : xs[k];
        const int64_t qb = q0 + q_in;
        const float* qs = scale + k * 32;
        const int count = queries - q_in < 32 ? queries - q_in : 32;
        if constexpr (WAY == kTma) {
          stage_queries<OT>(v, qs, row_scale, bias[k], out_buf, row_in_cta, grp, count, &tm_out,
                            static_cast<int>(row_cta), static_cast<int>(qb));
        } else if constexpr (WAY == kStaged) {
          ragged.store(v, qs, row_scale, bias[k], grp, count, out + qb * p.ldo + row_cta, p.ldo,
                       p.n - row_cta < kRows ? static_cast<int>(p.n - row_cta) : kRows);
        } else {
          constexpr bool PAIR = WAY == kPairs;
          // Lanes 2i and 2i + 1 trade 16-bit scores when these leave in pairs:
          // the even one stores both rows' of query j, the odd one of j + 1.
          const int odd = PAIR ? lane & 1 : 0;
          OT* o = out + (qb + odd) * p.ldo + (row - odd);
          if (row_warp + 32 <= p.n) {
            if (count == 32) {
              store_queries<OT, PAIR, 0>(v, qs, row_scale, bias[k], o, p.ldo, odd, 32);
            } else {
              store_queries<OT, PAIR, 1>(v, qs, row_scale, bias[k], o, p.ldo, odd, count);
            }
          } else {
            // The last base rows. keep: this lane's pair exists (2), or its
            // first row alone (1: the last of an odd count), or nothing (0).
            const int64_t left = p.n - (row - odd);
            store_ragged<OT, PAIR>(v, qs, row_scale, bias[k], o, p.ldo, odd, count,
                                   left >= 2 ? 2 : left < 0 ? 0 : static_cast<int>(left));
          }
        }
      }
      if (!freed) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_shared(tempty_bar(acc), 0));
      }
      if (++acc == p.accs) {
        acc = 0;
        acc_phase ^= 1;
      }
      fresh = advance(qg, bt);
    }
    if (WAY == kTma && quarter == 0 && lane == 0) store_wait();
  }

  if (warp == 1 && lane == 0) quiet_wait(done_bar, 0);
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 512);
  if (threadIdx.x == 0 && *s_abort) atomicOr(&g_int8_err, 1u);
}

template <typename OT, int WAY>
cudaError_t launch_typed(const CUtensorMap* maps, const Params& p, int clusters, size_t smem, cudaStream_t stream) {
  auto kern = int8_scores_kernel<OT, WAY>;
  // The limit belongs to the kernel, not to the launch: always the most, so that
  // a call on another thread with less shared memory leaves this one its own.
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemLimit));
  if (e != cudaSuccess) return e;
  return launch_after(kern, 2 * clusters, kThreads, smem, stream, maps[0], maps[1], maps[2], p);
}

template <typename OT>
cudaError_t launch_16(Way way, const CUtensorMap* maps, const Params& p, int clusters, size_t smem, cudaStream_t stream) {
  switch (way) {
    case kTma: return launch_typed<OT, kTma>(maps, p, clusters, smem, stream);
    case kStaged: return launch_typed<OT, kStaged>(maps, p, clusters, smem, stream);
    case kPairs: return launch_typed<OT, kPairs>(maps, p, clusters, smem, stream);
    default: return launch_typed<OT, kSingle>(maps, p, clusters, smem, stream);
  }
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
  // Few queries: several groups of 256 base rows per tile, as many as still
  // leave two tiles per cluster. Per tile of one slice and 32 queries the MMA
  // warp's waits and commits take about 1250 clocks, HBM 690.
  p.subs = p.n_cols <= 64 ? 4 : p.n_cols <= 128 ? 2 : 1;
  const int64_t size = a.type == kElemF32 ? 4 : 2;
  Way way = kSingle;
  if (reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.ldo * size % 16 == 0 && a.n * size % 16 == 0 &&
      a.ldo * size < (int64_t(1) << 40))
    way = kTma;
  else if (a.m * a.n * size >= kStagedBytes)
    way = kStaged;
  else if (size == 2 && reinterpret_cast<uintptr_t>(a.out) % 4 == 0 && a.ldo % 2 == 0)
    way = kPairs;
  while (p.subs > 1 && (a.n + p.subs * 2 * kRows - 1) / (p.subs * 2 * kRows) * groups < 2 * clusters) p.subs /= 2;
  p.base_tiles = static_cast<int>((a.n + p.subs * 2 * kRows - 1) / (p.subs * 2 * kRows));
  p.accs = p.subs * p.n_cols <= 128 ? 4 : 2;
  // A base that several query groups read, and that L2 (126 MB) can hold beside
  // what is being written, stays there; otherwise it goes first.
  p.keep_base = groups > 1 && a.n * a.d <= (int64_t(96) << 20);
  if (groups * p.base_tiles > 0x7fffffff) return cudaErrorInvalidValue;
  p.groups = static_cast<int>(groups);
  // Teams read the same base tiles at about the same time, so that the base
  // comes from HBM once per `teams` query groups; teams of eight clusters or
  // more write runs of 4 KB and more. The most of them that leave 95% of the
  // clusters busy.
  p.teams = 1;
  for (int64_t k = 2; k <= groups && 8 * k <= clusters; ++k) {
    const int64_t turns = (groups + k - 1) / k;
    if (groups * (clusters / k * k) * 100 >= 95 * turns * k * clusters) p.teams = static_cast<int>(k);
  }
  const int64_t per_team = (groups + p.teams - 1) / p.teams * p.base_tiles;
  p.width = clusters / p.teams;
  if (p.width > per_team) p.width = static_cast<int>(per_team);
  clusters = p.teams * p.width;
  p.kc = (a.d + kSlice - 1) / kSlice;
  const int b_slice = p.n_cols / 2 * kSlice;
  const size_t fixed = kFixed + kGroups * staging(way);
  // Resident queries leave 80 KB or more of ring: what HBM's latency times an
  // SM's share of the bandwidth asks for and half more.
  const int a_bytes = p.subs * kA;
  p.resident = fixed + static_cast<size_t>(p.kc) * b_slice + ((4 + p.subs) / p.subs) * a_bytes <= kSmemLimit;
  p.stage_bytes = p.resident ? a_bytes : a_bytes + b_slice;
  const size_t b_bytes = p.resident ? static_cast<size_t>(p.kc) * b_slice : 0;
  const int fit = static_cast<int>((kSmemLimit - fixed - b_bytes) / p.stage_bytes);
  p.stages = fit < kMaxStages ? fit : kMaxStages;
  const size_t smem = fixed + b_bytes + static_cast<size_t>(p.stages) * p.stage_bytes;
  CUtensorMap maps[3];
  cudaError_t e = encode_rows_map(&maps[0], kElemS8, a.x, a.d, a.n, a.ldx, kSlice, kRows, 128);
  if (e == cudaSuccess) e = encode_rows_map(&maps[1], kElemS8, a.q, a.d, a.m, a.ldq, kSlice, p.n_cols / 2, 128);
  if (e == cudaSuccess && way == kTma)
    e = encode_rows_map(&maps[2], a.type, a.out, a.n, a.m, a.ldo * size, kRows, size == 4 ? 16 : 32, 0);
  else
    maps[2] = maps[0];  // not used
  if (e != cudaSuccess) return e;
  switch (a.type) {
    case kElemF32:
      return way == kTma      ? launch_typed<float, kTma>(maps, p, clusters, smem, stream)
             : way == kStaged ? launch_typed<float, kStaged>(maps, p, clusters, smem, stream)
                              : launch_typed<float, kSingle>(maps, p, clusters, smem, stream);
    case kElemF16: return launch_16<__half>(way, maps, p, clusters, smem, stream);
    case kElemBf16: return launch_16<__nv_bfloat16>(way, maps, p, clusters, smem, stream);
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
