// Products of the dense feed-forward operators for sm_100a (see mmoe_dense.cuh).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mmoe_dense_device.cuh"
#include "mmoe_dense_rules.h"

namespace mmoe {

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Products on CTA pairs: a persistent pair takes tiles of 256 rows of A by 64 to 256 rows of B (tcgen05.mma.cta_group::2, M = 256), of
// which each CTA stages 128 rows of A and half of B, 128 bytes of K a stage.  One warp of the leader issues for both SMs; the
// accumulators of two tiles alternate in tensor memory, so that a tile's epilogue runs beside the next one's products.
// kGated: the leader stages gate rows and its peer the up rows of the same channels, so the two values of a channel are half a tile of
// columns apart in one lane.
// An operand whose rows run along K is staged as such; one that is stored transposed (k_rows) as 64 x 64 blocks with its own rows along the
// 128 bytes, which the tensor core reads just as well (MN-major descriptors): no transposed copy is made.
//
// What bounds it: a tile of 256 x 256 costs each tensor core 512 clk a stage and its SM 32 KB from the L2, at 55-60 bytes a clock, so both ends
// are near their limit there, and narrower tiles are bound by their copies (choose_cols).  Long calls sit at the power limit instead: 3840 tokens,
// 5120 x 2304, one launch at a time, at 1.48-1.67 GHz: 16-bit gated product 129 us (1.41 PFLOP/s, g and u written too), second product 64 (1.40),
// gradients 133 (dh with dw2, 1.37) and 226 (dx with dw13, 1.60; tensor pipe active 96 %); 8-bit gated product 60 (3.0), second 34 (2.6).
// A launch of one turn has 1.3-1.6 us in front of its first products and 1.2-4 us of epilogue behind its last.
// ---------------------------------------------------------------------------------------------------------------------
// One product of a launch
struct DensePart {
  CUtensorMap map_a, map_b;
  DenseEpilogue epi;
  int32_t m, n, k_stages;
  int32_t cols;              // rows of B per tile (kGated: half of them gate rows), a multiple of 32
  int32_t m_tiles, n_tiles;
  int32_t first_tile;        // of the launch
  int32_t kind, a_mn, b_mn;
  uint32_t idesc, tx_bytes;  // tx_bytes: a stage's copies into both CTAs
};

struct DenseParams {
  DensePart part[kMaxParts];
  int32_t parts, tiles;
  int32_t stages, stage_bytes;
  int32_t* status;
  int64_t timeout_ns;
};

struct PairControl {
  uint64_t full[kMaxStages];    // leader only: every copy of the stage, in both CTAs, has landed
  uint64_t empty[kMaxStages];   // issuer -> producers of both CTAs
  uint64_t acc_full[2];         // issuer -> epilogues of both CTAs
  uint64_t acc_empty[2];        // leader only: epilogue warps of both CTAs -> issuer
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};

static_assert(sizeof(PairControl) <= 1024, "control block");

// The t-th tile of a product: eight tiles of rows at a time, all columns of those before the next eight, so that what runs at once reads few
// different rows of either operand.
struct TilePlace {
  int m, n;
};
__device__ __forceinline__ TilePlace place_tile(const DensePart& q, int t) {
  t -= q.first_tile;
  const int group = t / (8 * q.n_tiles), first = group * 8, rows = min(8, q.m_tiles - first), in = t - group * 8 * q.n_tiles;
  return TilePlace{first + in % rows, in / rows};
}
template <int kParts>
__device__ __forceinline__ const DensePart& part_of(const DenseParams& p, int t) {
  return p.part[kParts > 1 && p.parts > 1 && t >= p.part[1].first_tile ? 1 : 0];
}

// A warp's 32 x 32 block of sums, turned from one row per lane to eight columns per lane.  16-byte piece g of row r lies at g ^ (r & 7).
__device__ __forceinline__ void block_write(uint8_t* block, int lane, const uint32_t (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    *reinterpret_cast<uint4*>(block + lane * 128 + ((g ^ (lane & 7)) << 4)) = make_uint4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
}
__device__ __forceinline__ void block_read8(const uint8_t* block, int row, int piece, float (&v)[8]) {
  const float4 lo = *reinterpret_cast<const float4*>(block + row * 128 + ((piece ^ (row & 7)) << 4));
  const float4 hi = *reinterpret_cast<const float4*>(block + row * 128 + (((piece + 1) ^ (row & 7)) << 4));
  v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
}

// f(whether A, whether B is staged with its rows along the 128 bytes), known to the compiler
template <bool kInt8, int kSet, typename F>
__device__ __forceinline__ void by_order(const DensePart& q, F f) {
  if (kInt8 || kSet == kGated || (kSet == kLinear && q.b_mn == 0)) f(std::false_type(), std::false_type());
  else if (q.a_mn == 0) f(std::false_type(), std::true_type());
  else f(std::true_type(), std::true_type());
}

// An epilogue warp's share of a tile: 32 of this CTA's 128 rows, every other block of columns.  A lane has a row of sums in tensor memory; a block
// of 32 x 32 of them is turned in shared memory, so that rows leave in 64 bytes and more.  Two warps to each quadrant instead of one:
// 8-bit second product of 3840 tokens 61 -> 35 us.
struct EpiPlace {
  uint32_t d;                // accumulator, this warp's lanes
  int row0, rows, col0, last;
  int side, lane;
  uint8_t* block;
};
template <bool kInt8, int kKind, typename Release>
__device__ __forceinline__ void pair_epilogue(const DenseEpilogue& epi, int cols, const EpiPlace& e, float row_scale, Release release) {
  constexpr int kChunk = kKind == kGated ? 16 : 32, kLanes = kChunk / 8, kRowsAtOnce = 32 / kLanes, kTurns = kLanes;
  const int sub = e.lane / kLanes, piece = e.lane % kLanes;
  const int chunks = e.rows > 0 ? (e.last - e.col0 + kChunk - 1) / kChunk : 0;
  if (e.side >= chunks) release();
#pragma unroll 1
  for (int c = e.side; c < chunks; c += 2) {
    const DenseFinish<kKind, kInt8> finish(epi, e.last, e.col0 + kChunk * c + 8 * piece);
    float g[kTurns][8], u[kTurns][8];
    if (kKind == kGatedGrad) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i)
        if (i * kRowsAtOnce + sub < e.rows) finish.fetch(e.row0 + i * kRowsAtOnce + sub, g[i], u[i]);
    }
    uint32_t v[32];
    if (kKind == kGated) {
      tc_ld16(e.d + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(v));
      tc_ld16(e.d + cols / 2 + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
    } else {
      tc_ld32(e.d + 32 * c, v);
    }
    tc_ld_wait();
    if (kInt8) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(static_cast<float>(static_cast<int32_t>(v[j])));
    }
    if (c + 2 >= chunks) release();
    __syncwarp();                             // the previous block has been read
    block_write(e.block, e.lane, v);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int r = i * kRowsAtOnce + sub;
      float a[8];
      block_read8(e.block, r, 2 * piece, a);
      if (kKind == kGated) block_read8(e.block, r, 4 + 2 * piece, g[i]);
      const float rs = kInt8 ? __shfl_sync(0xffffffffu, row_scale, r) : 0.f;
      if (r < e.rows) finish.row(e.row0 + r, rs, a, g[i], u[i]);
    }
  }
}

// kSet: the kind of every product of the launch; kGatedGrad: of the first or none, the others kLinear.  kParts: most products; with one, its
// fields are at fixed places (two: 8-bit projection of 777 tokens 23.7 -> 24.7 us, 16-bit block of 1021 57.5 -> 58.5).
template <bool kInt8, int kSet, int kParts>
__global__ void __launch_bounds__(kPairThreads, 1) dense_pair_kernel(const __grid_constant__ DenseParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in both CTAs
  PairControl* ctl = reinterpret_cast<PairControl*>(smem);
  uint8_t* blocks = smem + 1024;
  uint8_t* stages = blocks + kEpiWarps * kEpiBlock;
  constexpr int kDepth = kInt8 ? 128 : 64;              // k's per stage

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.parts; ++i) {
      prefetch_map(&p.part[i].map_a);
      prefetch_map(&p.part[i].map_b);
    }
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&ctl->full[i]), 1);
      mbar_init(smem_u32(&ctl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[i]), 2 * kEpiWarps);
    }
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // the peer's barriers are initialised before anything arrives on them
  tc_fence_after();
  chain_wait();                             // nothing above touches global memory
  chain_release();                          // in this order: what precedes this launch is complete when the next one starts
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  const int tiles = p.tiles, step = gridDim.x / 2, n_stages = p.stages;
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusDense, warp}, p.timeout_ns};
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);

  if (warp == 0) {
    // --------------------------------------------------------------------------------------------- producer
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t leader_full0 = map_to_cta(full0, 0), base = smem_u32(stages);
    bool ok = true;
    for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
      const DensePart& q = part_of<kParts>(p, t);
      const TilePlace at = place_tile(q, t);
      const int half = q.cols / 2, k_stages = q.k_stages;
      const uint32_t tx = q.tx_bytes;
      const int a_row = at.m * 2 * kPairRows + static_cast<int>(cta) * kPairRows;
      const int b_row = kSet == kGated ? at.n * half + static_cast<int>(cta) * q.epi.inter : at.n * q.cols + static_cast<int>(cta) * half;
      by_order<kInt8, kSet>(q, [&](auto a_order, auto b_order) {
        constexpr bool a_mn = decltype(a_order)::value, b_mn = decltype(b_order)::value;
        for (int kb = 0; kb < k_stages; ++kb) {
          if (!waiter.wait_uniform(empty0 + 8 * stage, phase ^ 1u)) { ok = false; break; }
          const uint32_t bar = leader_full0 + 8 * stage, a = base + stage * p.stage_bytes, b = a + kStageA;
          if (elect_one()) {
            if (cta == 0) mbar_expect_tx(full0 + 8 * stage, tx);
            if (a_mn) {
              pair_load_2d(a, &q.map_a, a_row, kb * kDepth, bar);
              pair_load_2d(a + 8192, &q.map_a, a_row + 64, kb * kDepth, bar);
            } else {
              pair_load_2d(a, &q.map_a, kb * kDepth, a_row, bar);
            }
            if (b_mn) {
              pair_load_2d(b, &q.map_b, b_row, kb * kDepth, bar);
              if (half > 64) pair_load_2d(b + 8192, &q.map_b, b_row + 64, kb * kDepth, bar);
            } else {
              pair_load_2d(b, &q.map_b, kb * kDepth, b_row, bar);
            }
          }
          __syncwarp();
          if (++stage == n_stages) { stage = 0; phase ^= 1u; }
        }
      });
    }
  } else if (warp == 1) {
    // --------------------------------------------------------------------------------------------- issuer
    if (cta == 0) {
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = true;
      const uint32_t lo0 = (smem_u32(stages) & 0x3FFFFu) >> 4, lo_step = p.stage_bytes >> 4;
      for (int t = blockIdx.x / 2; ok && t < tiles; t += step, ++it) {
        const DensePart& q = part_of<kParts>(p, t);
        const uint32_t idesc = q.idesc;
        const int k_stages = q.k_stages;
        const uint32_t acc = it & 1u, d = tmem_base + acc * kPairCols;
        if (!waiter.wait_uniform(smem_u32(&ctl->acc_empty[acc]), ((it >> 1) & 1u) ^ 1u)) break;
        tc_fence_after();
        by_order<kInt8, kSet>(q, [&](auto a_order, auto b_order) {
          constexpr bool a_mn = decltype(a_order)::value, b_mn = decltype(b_order)::value;
          const uint64_t a_hi = operand_desc(a_mn, 8192), b_hi = operand_desc(b_mn, 8192);
          // a K of 32 bytes further: along the 128 bytes, or 16 rows of them
          constexpr uint32_t kStepA = a_mn ? 2048 >> 4 : 2, kStepB = b_mn ? 2048 >> 4 : 2;
          for (int kb = 0; kb < k_stages; ++kb) {
            if (!waiter.wait_uniform(full0 + 8 * stage, phase)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a = lo0 + stage * lo_step, b = a + (kStageA >> 4);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                pair_product<kInt8>(d, a_hi | (a + kStepA * k), b_hi | (b + kStepB * k), idesc, (kb | k) != 0 ? 1u : 0u);
              pair_commit(empty0 + 8 * stage);
            }
            __syncwarp();
            if (++stage == n_stages) { stage = 0; phase ^= 1u; }
          }
        });
        if (ok && elect_one()) pair_commit(smem_u32(&ctl->acc_full[acc]));
        __syncwarp();
      }
    }
  } else {
    // --------------------------------------------------------------------------------------------- epilogue
    const int quadrant = warp & 3;                    // of the TMEM lanes: the one this warp may read
    const uint32_t leader_empty = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    EpiPlace e;
    e.side = (warp - 2) >> 2, e.lane = lane, e.block = blocks + (warp - 2) * kEpiBlock;
    uint32_t it = 0;
    for (int t = blockIdx.x / 2; t < tiles; t += step, ++it) {
      const DensePart& q = part_of<kParts>(p, t);
      const DenseEpilogue epi = q.epi;
      const TilePlace at = place_tile(q, t);
      const uint32_t acc = it & 1u;
      const int width = kSet == kGated ? q.cols / 2 : q.cols;
      e.row0 = at.m * 2 * kPairRows + static_cast<int>(cta) * kPairRows + quadrant * 32, e.rows = min(32, q.m - e.row0);
      e.col0 = at.n * width, e.last = min(q.n, e.col0 + width);
      e.d = tmem_base + acc * kPairCols + (static_cast<uint32_t>(quadrant * 32) << 16);
      const float row_scale = kInt8 && lane < e.rows ? epi.row_scale[e.row0 + lane] : 0.f;
      if (kSet == kGatedGrad && q.kind == kGatedGrad && e.side == 0 && lane < e.rows) {
        // g and u come from HBM, a row's 1 KB each by now
        const float* keep = epi.preact + (int64_t)(e.row0 + lane) * 2 * epi.inter + e.col0;
        prefetch_bulk(keep, (e.last - e.col0) * 4);
        prefetch_bulk(keep + epi.inter, (e.last - e.col0) * 4);
      }
      if (!waiter.wait_warp(smem_u32(&ctl->acc_full[acc]), (it >> 1) & 1u, q.k_stages)) break;
      tc_fence_after();
      const auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(leader_empty + 8 * acc);
      };
      if (kSet == kGatedGrad && q.kind == kLinear) pair_epilogue<kInt8, kLinear>(epi, q.cols, e, row_scale, release);
      else pair_epilogue<kInt8, kSet>(epi, q.cols, e, row_scale, release);
    }
  }

  // ---------------------------------------------------------------------------------------------------- teardown
  __syncwarp();
  if (ctl->abort_flag != 0) {               // copies still in flight land before this CTA's shared memory goes
    const uint64_t t0 = global_timer();
    while (global_timer() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // no CTA leaves while its peer may still arrive on its barriers
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// Products of few tokens, bound by the bytes of B (the weights): 128 of its rows are operand A of the tensor core and the tokens, padded to 16,
// operand B, so that few tokens cost little.  kGated: 64 gate and 64 up rows.  K is split over the CTAs of a cluster, whose partial sums meet
// in shared memory, added in the order of the CTAs: no atomics, no workspace, and the same bits in every call.  They are sent in one copy to each
// CTA; read by every thread from the others' shared memory instead, 64 tokens of the block took 22.5 us, stored there value by value 23.7.
// One token, weights from HBM, replayed back to back: 8-bit 5120 x 4608 (23.6 MB) 7.4 us, 2304 x 5120 (11.8 MB) 5.4, 16-bit block (71 MB, two
// launches) 17.9; 64 tokens 9.0, 7.0 and 21.2.  Of the 7.4: 2.3 until the first stage has come, 3.6 at 6.5 TB/s, 1-2 for the sums and the last CTAs.
// The second product's weights requested ahead of its wait, beside the first product: 18.1 -> 19.8, so it does not.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = 128;                         // rows of B per tile
constexpr int kFewThreads = 256;
constexpr int kFewMaxStages = 10;                      // what fits beside 48 tokens; fewer tokens have half of an SM
constexpr int kFewTokens = 160, kFewMaxTokens = 192;  // with the weights as they are stored; read along their rows (dense_few_tokens)
constexpr int kFewMaxSplit = 8;
constexpr int kFewSmem = 227 * 1024;
constexpr int kFewControl = 2048, kFewApart = kFewControl + 1024;      // beside the stages: control block, and the slack for aligning the base
// Half of an SM for each CTA: up to so many tokens, which need no more, so that the next launch's CTAs find room; and where there are more tiles than
// SMs, so that one CTA's start and sums run beside another's products: 8-bit projection, 2304 x 20000, one token 14.7 -> 10.2 us, 128
// tokens 19.7 -> 14.8; 5120 x 25000 27.4 -> 23.1 and 34.1 -> 28.9; 5120 x 152064, 1, 64 and 128 tokens 117 -> 116, 133 -> 137, 168 -> 154 (the
// one there that loses, 3 %, between two that gain).  With 128 tiles, 8192 x 16384, 64 tokens 26.2 -> 29.4, so not there.
constexpr int kFewSmemHalf = 113 * 1024;
constexpr int kFewHalfTokens = 32;

struct FewParams {
  CUtensorMap map_w, map_t;
  int32_t m, n, k_stages;
  int32_t tokens;            // m, rounded up to 16
  int32_t split;             // CTAs of a cluster
  int32_t stages;
  uint32_t idesc;
  int32_t tmem_cols;
  DenseEpilogue epi;
  int32_t* status;
  int64_t timeout_ns;
};

struct FewControl {
  uint64_t full[kFewMaxStages], empty[kFewMaxStages];
  uint64_t acc_full;
  uint64_t sums_in;             // what the other CTAs of the cluster send
  uint32_t tmem_base;
  volatile int32_t abort_flag;
  float row_scale[kFewMaxTokens];
};
static_assert(sizeof(FewControl) <= kFewControl, "control block");
// sums of m tokens, padded to 16, and what the other CTAs send of those that this one finishes
constexpr int few_sum_bytes(int m, int split) { return ((m + 15) / 16 * 16 + (split - 1) * ((m + split - 1) / split)) * kFewRows * 4; }
static_assert((kFewSmem - kFewApart) / (kFewRows * 128 + (kFewHalfTokens + 16) * 128) == kFewMaxStages &&
              (kFewSmemHalf - kFewApart) / (kFewRows * 128 + 16 * 128) <= kFewMaxStages, "stages of few tokens");
static_assert(few_sum_bytes(kFewMaxTokens, 1) <= kFewSmem - kFewApart, "partial sums of a tile fit where the stages were");

// adds eight neighbouring sums; `swap`: second half first, so that eight lanes read all banks
template <bool kInt8>
__device__ __forceinline__ void add_part(const uint8_t* at, bool swap, float (&v)[8], int32_t (&whole)[8]) {
  const float4 p = *reinterpret_cast<const float4*>(at + (swap ? 16 : 0)), q = *reinterpret_cast<const float4*>(at + (swap ? 0 : 16));
  const float4 lo = swap ? q : p, hi = swap ? p : q;
  const float part[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (kInt8) whole[j] += __float_as_int(part[j]);
    else v[j] += part[j];
  }
}

template <bool kInt8, bool kWmn, int kKind>
__global__ void __launch_bounds__(kFewThreads, 1) dense_few_kernel(const __grid_constant__ FewParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in all CTAs
  FewControl* ctl = reinterpret_cast<FewControl*>(smem);
  uint8_t* stages = smem + kFewControl;
  constexpr int kDepth = kInt8 ? 128 : 64;
  constexpr int kWBytes = kFewRows * 128;
  const int stage_bytes = kWBytes + p.tokens * 128;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / p.split;
  const int k0 = static_cast<int>((int64_t)p.k_stages * rank / p.split), k1 = static_cast<int>((int64_t)p.k_stages * (rank + 1) / p.split);
  if (threadIdx.x == 0) {
    prefetch_map(&p.map_w);
    prefetch_map(&p.map_t);
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&ctl->full[i]), 1);
      mbar_init(smem_u32(&ctl->empty[i]), 1);
    }
    mbar_init(smem_u32(&ctl->acc_full), 1);
    mbar_init(smem_u32(&ctl->sums_in), 1);
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]), base = smem_u32(stages);
  const int n_stages = p.stages;
  chain_wait();                             // nothing above touches global memory
  chain_release();                          // in this order: what precedes this launch is complete when the next one starts
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusDense + 1, warp}, p.timeout_ns};

  if (warp == 0) {
    // --------------------------------------------------------------------------------------------- producer
    int stage = 0;
    uint32_t phase = 0;
    const int w_row = tile * (kKind == kGated ? kFewRows / 2 : kFewRows);
    for (int kb = k0; kb < k1; ++kb) {
      if (!waiter.wait_uniform(empty0 + 8 * stage, phase ^ 1u)) break;
      const uint32_t bar = full0 + 8 * stage, w = base + stage * stage_bytes;
      if (elect_one()) {
        mbar_expect_tx(bar, stage_bytes);
        if (kKind == kGated) {
          tma_load_2d(w, &p.map_w, kb * kDepth, w_row, bar);
          tma_load_2d(w + 8192, &p.map_w, kb * kDepth, p.epi.inter + w_row, bar);
        } else if (kWmn) {
          tma_load_2d(w, &p.map_w, w_row, kb * kDepth, bar);
          tma_load_2d(w + 8192, &p.map_w, w_row + 64, kb * kDepth, bar);
        } else {
          tma_load_2d(w, &p.map_w, kb * kDepth, w_row, bar);
        }
        tma_load_2d(w + kWBytes, &p.map_t, kb * kDepth, 0, bar);
      }
      __syncwarp();
      if (++stage == n_stages) { stage = 0; phase ^= 1u; }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------------------------------------------- issuer
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint64_t w_hi = operand_desc(kWmn, 8192), t_hi = operand_desc(false, 0);
    constexpr uint32_t kStepW = kWmn ? 2048 >> 4 : 2;
    for (int kb = k0; kb < k1; ++kb) {
      if (!waiter.wait_uniform(full0 + 8 * stage, phase)) { ok = false; break; }
      tc_fence_after();
      const uint32_t w = ((base + stage * stage_bytes) & 0x3FFFFu) >> 4, t = w + (kWBytes >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) single_product<kInt8>(tmem_base, w_hi | (w + kStepW * k), t_hi | (t + 2 * k), p.idesc, kb > k0 || k > 0 ? 1u : 0u);
        tc_commit(empty0 + 8 * stage);
      }
      __syncwarp();
      if (++stage == n_stages) { stage = 0; phase ^= 1u; }
    }
    if (ok && elect_one()) tc_commit(smem_u32(&ctl->acc_full));
    __syncwarp();
  }

  // ------------------------------------------------------------------------------------------------- sums
  // A thread finishes the same eight channels of every so many tokens; what belongs to the channels and tokens is fetched ahead.
  constexpr int kGroups = kKind == kGated ? kFewRows / 16 : kFewRows / 8;     // eight channels each
  static_assert(kFewThreads % kGroups == 0, "a thread keeps its channels");
  const int tokens = p.m, g = static_cast<int>(threadIdx.x) % kGroups;
  const DenseFinish<kKind, kInt8> finish(p.epi, p.n, tile * 8 * kGroups + 8 * g);
  if (kInt8)
    for (int t = threadIdx.x; t < tokens; t += kFewThreads) ctl->row_scale[t] = p.epi.row_scale[t];
  // The partial sums take the place of the stages, which this CTA needs no more when its accumulator is complete: [token][128 rows].  Each CTA
  // of the cluster finishes some of the tokens; the others send it theirs, in one copy each, when no CTA needs its stages any more.
  constexpr int kRowBytes = kFewRows * 4;
  const int own = (tokens + p.split - 1) / p.split, first = rank * own, mine = max(0, min(own, tokens - first));
  const uint32_t came = smem_u32(&ctl->sums_in);
  uint8_t* sent = stages + p.tokens * kRowBytes;       // [CTA, this one left out][token][128 rows]
  if (p.split > 1 && threadIdx.x == 0) mbar_expect_tx(came, (p.split - 1) * mine * kRowBytes);
  if (warp >= 2 && warp < 6 && waiter.wait_warp(smem_u32(&ctl->acc_full), 0, k1 - k0)) {
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;
    const uint32_t d = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    for (int j0 = 0; j0 < tokens; j0 += 16) {
      uint32_t v[16];
      tc_ld16(d + j0, v);
      tc_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) reinterpret_cast<uint32_t*>(stages)[(j0 + j) * kFewRows + row] = v[j];
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  cluster_sync_all();
  if (p.split > 1) {
    if (threadIdx.x == 0)
      for (int r = 0; r < p.split; ++r) {
        const int theirs = min(own, tokens - r * own);
        if (r != rank && theirs > 0)
          cluster_send(map_to_cta(base + (p.tokens + (rank < r ? rank : rank - 1) * own) * kRowBytes, r), base + r * own * kRowBytes, theirs * kRowBytes, map_to_cta(came, r));
      }
    __syncwarp();
    waiter.wait_warp(came, 0, 0);
    __syncwarp();
    cluster_arrive();                       // what this CTA waited for has come; behind the matching wait, all that it has sent has
  }
#pragma unroll 2
  for (int i = threadIdx.x; i < mine * kGroups; i += kFewThreads) {
    const int t = i / kGroups, at = (t * kFewRows + 8 * g) * 4;
    const bool swap = (g & 4) != 0;
    float a[8] = {}, b[8] = {}, u[8];
    int32_t wa[8] = {}, wb[8] = {};
    if (kKind == kGatedGrad) finish.fetch(first + t, b, u);
#pragma unroll 4
    for (int r = 0; r < p.split; ++r) {                // in the order of the CTAs
      const uint8_t* from = (r == rank ? stages + first * kRowBytes : sent + (r < rank ? r : r - 1) * own * kRowBytes) + at;
      add_part<kInt8>(from, swap, a, wa);
      if (kKind == kGated) add_part<kInt8>(from + kRowBytes / 2, swap, b, wb);
    }
    if (kInt8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] = static_cast<float>(wa[j]), b[j] = static_cast<float>(wb[j]);
    }
    finish.row(first + t, kInt8 ? ctl->row_scale[first + t] : 0.f, a, b, u);
  }
  if (p.split > 1) {
    __syncwarp();
    cluster_wait();
  }

  // ---------------------------------------------------------------------------------------------------- teardown
  if (ctl->abort_flag != 0) {
    const uint64_t t0 = global_timer();
    while (global_timer() - t0 < 200000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.tmem_cols) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
std::atomic<EncodeFn> g_encode{nullptr};
std::atomic<int> g_sms[kMaxDevices];        // per device, 0: prepare_dense() has not run there

// `rows` x k matrix; boxes of 128 bytes of K by `box` rows, or (stored transposed) of 64 rows by 64 k's
bool encode(CUtensorMap* map, const DenseOperand& o, int type, uint64_t rows, uint64_t k, uint32_t box) {
  const uint64_t size = type == kDenseInt8 ? 1 : 2;
  const cuuint64_t dims[2] = {o.k_rows ? rows : k, o.k_rows ? k : rows};
  const cuuint64_t strides[1] = {static_cast<uint64_t>(o.ld) * size};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(128 / size), o.k_rows ? 64u : box};
  const cuuint32_t one[2] = {1, 1};
  const CUtensorMapDataType t = type == kDenseInt8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == kDenseBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return g_encode.load()(map, t, 2, const_cast<void*>(o.p), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename F>
cudaError_t for_each_pair_kernel(F f) {
  cudaError_t e = f(dense_pair_kernel<false, kGated, 1>, false, kGated, 1);
  if (e == cudaSuccess) e = f(dense_pair_kernel<false, kLinear, 1>, false, kLinear, 1);
  if (e == cudaSuccess) e = f(dense_pair_kernel<false, kLinear, 2>, false, kLinear, 2);
  if (e == cudaSuccess) e = f(dense_pair_kernel<false, kGatedGrad, 1>, false, kGatedGrad, 1);
  if (e == cudaSuccess) e = f(dense_pair_kernel<false, kGatedGrad, 2>, false, kGatedGrad, 2);
  if (e == cudaSuccess) e = f(dense_pair_kernel<true, kGated, 1>, true, kGated, 1);
  if (e == cudaSuccess) e = f(dense_pair_kernel<true, kLinear, 1>, true, kLinear, 1);
  return e;
}

template <typename F>
cudaError_t for_each_few_kernel(F f) {
  cudaError_t e = f(dense_few_kernel<false, false, kGated>, kDenseBf16, false, kGated);
  if (e == cudaSuccess) e = f(dense_few_kernel<false, false, kLinear>, kDenseBf16, false, kLinear);
  if (e == cudaSuccess) e = f(dense_few_kernel<false, true, kGatedGrad>, kDenseBf16, true, kGatedGrad);
  if (e == cudaSuccess) e = f(dense_few_kernel<false, true, kLinear>, kDenseBf16, true, kLinear);
  if (e == cudaSuccess) e = f(dense_few_kernel<true, false, kGated>, kDenseInt8, false, kGated);
  if (e == cudaSuccess) e = f(dense_few_kernel<true, false, kLinear>, kDenseInt8, false, kLinear);
  return e;
}

std::atomic<int> g_clusters[kMaxDevices][kFewMaxSplit + 1];     // clusters of so many CTAs that run at once

cudaError_t launch_few(const DenseProduct& p, int sms, cudaStream_t s) {
  FewParams d;
  d.m = p.m, d.n = p.n;
  const int depth = p.type == kDenseInt8 ? 128 : 64;
  d.k_stages = (p.k + depth - 1) / depth;
  d.tokens = (p.m + 15) & ~15;
  const int width = p.kind == kGated ? kFewRows / 2 : kFewRows, tiles = (p.n + width - 1) / width;
  const bool halves = d.tokens <= kFewHalfTokens || (tiles > sms && few_sum_bytes(p.m, 1) <= kFewSmemHalf - kFewApart);
  const int smem = halves ? kFewSmemHalf : kFewSmem;
  d.stages = std::min((smem - kFewApart) / (kFewRows * 128 + d.tokens * 128), kFewMaxStages);
  // CTAs that share a tile's K: what a stage costs each of them, or the weights' bytes all, against what meeting costs, in clocks.  With 1, 2, 3, 4
  // of them (- : do not fit at once), 8-bit gated product 5120 x 4608: one token 10.3, 8.0, 7.5, 7.4 us, 16 tokens 10.5, 8.3, 7.8, 7.9, 64 tokens
  // 11.6, 8.95, 8.98, - , 128 tokens 13.2, 10.6, 11.1, - ; second product 2304 x 5120, one token 6.3, 5.55, 5.4, - , 32 tokens 7.2, 6.3, 5.9, - , 128
  // tokens 9.15, 8.3, 9.0, - ; 16-bit block, one token 27.7, 19.8, 17.9, 17.6, 64 tokens 29.7, 21.9, 21.1, - , 144 tokens 35.4, 27.3, 25.9, - .  It takes
  // 3 where the weights' bytes are the cost, 2 in the second product from 16 tokens on; at most 0.5 us from the best (128 tokens, gated).
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t from_hbm = (int64_t)p.n * (p.kind == kGated ? 2 : 1) * d.k_stages * 128 / 4450;
  int64_t least = INT64_MAX;
  d.split = 1;
  for (int c = 1; c <= kFewMaxSplit; ++c) {
    const bool at_once = halves ? (int64_t)tiles * c <= sms : tiles <= g_clusters[dev][c].load();
    if (c > 1 && (!at_once || d.k_stages < 2 * c || few_sum_bytes(p.m, c) > smem - kFewApart)) continue;
    const int64_t cost = std::max(from_hbm, (int64_t)(d.k_stages + c - 1) / c * (300 + d.tokens)) + (int64_t)c * 20 * p.m;
    if (cost < least) least = cost, d.split = c;
  }
  d.idesc = product_idesc(p.type, p.b.k_rows, false, kFewRows, d.tokens);
  d.tmem_cols = d.tokens <= 32 ? 32 : d.tokens <= 64 ? 64 : d.tokens <= 128 ? 128 : 256;
  d.epi = p.epi;
  d.status = p.status;
  d.timeout_ns = (p.timeout_ms > 0 ? (int64_t)p.timeout_ms : 2000) * 1000000ll;
  if (!encode(&d.map_w, p.b, p.type, p.kind == kGated ? 2 * (uint64_t)p.n : p.n, p.k, width) || !encode(&d.map_t, p.a, p.type, p.m, p.k, d.tokens))
    return cudaErrorInvalidValue;
  bool found = false;
  const cudaError_t e = for_each_few_kernel([&](auto kernel, int type, bool w_mn, int kind) {
    if ((type == kDenseInt8) != (p.type == kDenseInt8) || w_mn != p.b.k_rows || kind != p.kind) return cudaSuccess;
    found = true;
    return launch_clustered(kernel, dim3(tiles * d.split), dim3(kFewThreads), smem, d.split, s, d);
  });
  return found ? e : cudaErrorInvalidValue;
}

cudaError_t launch_pairs(const DenseProduct* p, int parts, int sms, cudaStream_t s) {
  DenseParams d = {};
  int cols[kMaxParts] = {};
  choose_cols(p, parts, sms / 2, cols);
  d.parts = parts;
  d.status = p->status;
  d.timeout_ns = (p->timeout_ms > 0 ? (int64_t)p->timeout_ms : 2000) * 1000000ll;
  int64_t tiles = 0;
  const int set = p->kind;
  for (int i = 0; i < parts; ++i) {
    const DenseProduct& f = p[i];
    DensePart& q = d.part[i];
    if (f.a.k_rows && !f.b.k_rows) return cudaErrorInvalidValue;       // no caller has that
    if (i > 0 && (f.kind != kLinear || f.type == kDenseInt8 || f.type != p->type || set == kGated)) return cudaErrorInvalidValue;
    const int depth = f.type == kDenseInt8 ? 128 : 64, width = f.kind == kGated ? cols[i] / 2 : cols[i];
    q.epi = f.epi;
    q.m = f.m, q.n = f.n, q.cols = cols[i], q.kind = f.kind;
    q.a_mn = f.a.k_rows, q.b_mn = f.b.k_rows;
    q.k_stages = (f.k + depth - 1) / depth;
    q.m_tiles = (f.m + 2 * kPairRows - 1) / (2 * kPairRows);
    q.n_tiles = (f.n + width - 1) / width;
    q.first_tile = static_cast<int32_t>(tiles);
    tiles += (int64_t)q.m_tiles * q.n_tiles;
    if (tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
    q.idesc = product_idesc(f.type, f.a.k_rows, f.b.k_rows, 2 * kPairRows, cols[i]);
    const int bytes = kStageA + stage_b_bytes(f, cols[i]);
    q.tx_bytes = 2 * bytes;
    d.stage_bytes = std::max(d.stage_bytes, bytes);
    if (!encode(&q.map_a, f.a, f.type, f.m, f.k, kPairRows) || !encode(&q.map_b, f.b, f.type, f.kind == kGated ? 2 * (uint64_t)f.n : f.n, f.k, cols[i] / 2))
      return cudaErrorInvalidValue;
  }
  d.tiles = static_cast<int32_t>(tiles);
  d.stages = std::min(kPairStageRoom / d.stage_bytes, kMaxStages);
  const int grid = 2 * static_cast<int>(std::min<int64_t>(sms / 2, tiles));
  return for_each_pair_kernel([&](auto kernel, bool int8, int kind, int most) {
    if (int8 != (p->type == kDenseInt8) || kind != set || most != parts) return cudaSuccess;
    return launch_clustered(kernel, dim3(grid), dim3(kPairThreads), kPairSmem, 2, s, d);
  });
}

// ---------------------------------------------------------------------------------------------------------------------
// Per-token quantiser: s = max|x| / 127, q = x / s rounded to the nearest whole number, ties to even.
// A block per token; the row stays in registers between the two passes as far as it fits, so a value is read once: 3840 x 2304 (26 MB) 7.1 us,
// 3840 x 5120 (59 MB) 12.0, 20000 x 1024 12.9, 4.9 TB/s: the latency of the two passes; up to 64 rows 2.3, the launch.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 512, kQuantManyTokens = 512;
constexpr int kQuantHeld = 5;               // vectors that a thread keeps.  3840 x 5120 with 3, 5, 8, 12: 15.6, 11.5, 12.0, 14.5 us

// x / s as whole numbers, exactly, in the low bytes.  Adding 1.5 * 2^23 rounds the product with the reciprocal to a whole number q, the nearest
// one or, next to a border, its neighbour.  The remainder x - q s is exact in one fma (x has at most 11 bits and is above s / 2 in magnitude
// where it matters) and tells which; that is looked at once for all n values.  kTiny: s is so small that its reciprocal overflows or half of
// it is no number.
template <bool kTiny, int n>
__device__ __forceinline__ void quantize_some(const float (&x)[n], float s, float inv, uint32_t (&q)[n]) {
  constexpr float kShift = 12582912.f;
  float r[n], worst = 0.f;
#pragma unroll
  for (int j = 0; j < n; ++j) {
    const float shifted = kTiny ? __fadd_rn(__fdiv_rn(x[j], s), kShift) : fmaf(x[j], inv, kShift);
    q[j] = __float_as_uint(shifted);
    r[j] = fmaf(-__fsub_rn(shifted, kShift), s, x[j]);
    worst = fmaxf(worst, fabsf(r[j]));
  }
  if (kTiny ? worst + worst < s : worst < 0.5f * s) return;
#pragma unroll
  for (int j = 0; j < n; ++j) {
    const float twice = fabsf(r[j] + r[j]);
    if (twice > s || (twice == s && (q[j] & 1u) != 0)) q[j] += r[j] > 0.f ? 1u : ~0u;
  }
}

__device__ __forceinline__ __half2 pair_abs_max(__half2 top, __half2 v) { return __hmax2_nan(top, __habs2(v)); }
__device__ __forceinline__ __nv_bfloat162 pair_abs_max(__nv_bfloat162 top, __nv_bfloat162 v) { return __hmax2_nan(top, __habs2(v)); }
__device__ __forceinline__ float2 pair_floats(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 pair_floats(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <typename T> struct PairOf;
template <> struct PairOf<__half> { using type = __half2; };
template <> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };

// kVec: eight values at a time, else (widths, strides or places that do not allow it) one.  kWarps: a warp per token, eight of them to a block.
template <typename T, bool kVec, bool kWarps>
__global__ void __launch_bounds__(kQuantThreads) quantize_int8_kernel(const T* x, int64_t ld, int8_t* q, float* scales, int m, int k) {
  chain_wait();
  chain_release();
  using P = typename PairOf<T>::type;
  constexpr int kWide = kVec ? 8 : 1;
  struct alignas(sizeof(T) * kWide) Vec { T v[kWide]; };
  const int64_t row = kWarps ? blockIdx.x * 8 + threadIdx.y : blockIdx.x;
  if (row >= m) return;                     // a whole warp
  const Vec* in = reinterpret_cast<const Vec*>(x + row * ld);
  const int n = k / kWide, step = blockDim.x;
  Vec held[kQuantHeld];
  P top = {T(0.f), T(0.f)};
  const auto look = [&](const Vec& v) {
    if (kVec) {
#pragma unroll
      for (int j = 0; j < kWide / 2; ++j) top = pair_abs_max(top, reinterpret_cast<const P*>(&v)[j]);
    } else {
      top = pair_abs_max(top, P{v.v[0], T(0.f)});
    }
  };
#pragma unroll
  for (int i = 0; i < kQuantHeld; ++i) {
    const int at = threadIdx.x + i * step;
    if (at < n) held[i] = in[at];
  }
#pragma unroll
  for (int i = 0; i < kQuantHeld; ++i)
    if (threadIdx.x + i * step < n) look(held[i]);
  for (int at = threadIdx.x + kQuantHeld * step; at < n; at += step) look(in[at]);
  // magnitudes as bits: NaN is above infinity there, so neither is lost
  __shared__ uint32_t tops[kQuantThreads / 32];
  const float2 both = pair_floats(top);
  uint32_t bits = __reduce_max_sync(0xffffffffu, max(__float_as_uint(both.x), __float_as_uint(both.y)));
  if (!kWarps) {
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = bits;
    __syncthreads();
    for (int w = 0; w < (step >> 5); ++w) bits = max(bits, tops[w]);
  }
  const bool finite = bits < 0x7f800000u;
  const float s = !finite ? __uint_as_float(0x7fffffffu) : (bits == 0 ? 1.f : __fdiv_rn(__uint_as_float(bits), 127.f));
  if (threadIdx.x == 0) scales[row] = s;
  const auto finish = [&](auto some) {
    const auto put = [&](const Vec& v, int at) {
      float f[kWide];
      uint32_t b[kWide];
      if constexpr (kVec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 two = pair_floats(reinterpret_cast<const P*>(&v)[j]);
          f[2 * j] = two.x, f[2 * j + 1] = two.y;
        }
        some(f, b);
        uint2 o;
        o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
        reinterpret_cast<uint2*>(q + row * k)[at] = o;
      } else {
        f[0] = static_cast<float>(v.v[0]);
        some(f, b);
        q[row * k + at] = static_cast<int8_t>(b[0] & 0xffu);
      }
    };
#pragma unroll
    for (int i = 0; i < kQuantHeld; ++i) {
      const int at = threadIdx.x + i * step;
      if (at < n) put(held[i], at);
    }
    for (int at = threadIdx.x + kQuantHeld * step; at < n; at += step) put(in[at], at);
  };
  const float inv = __fdiv_rn(1.f, s);
  if (!finite) finish([](const float (&)[kWide], uint32_t (&b)[kWide]) { for (uint32_t& v : b) v = 0; });
  else if (s >= 0x1p-100f) finish([&](const float (&f)[kWide], uint32_t (&b)[kWide]) { quantize_some<false>(f, s, inv, b); });
  else finish([&](const float (&f)[kWide], uint32_t (&b)[kWide]) { quantize_some<true>(f, s, inv, b); });
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t ld, int8_t* q, float* scales, int m, int k, cudaStream_t s) {
  const T* in = static_cast<const T*>(x);
  const bool vec = k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  // Many tokens: as few threads as keep a row, so that many rows are on their way at once; few tokens: many, for a short way.
  const int n = vec ? k / 8 : k, most = m >= kQuantManyTokens ? std::max(32, std::min(kQuantThreads, (n + kQuantHeld - 1) / kQuantHeld)) : kQuantThreads;
  const int each = (n + most - 1) / most, threads = std::min(kQuantThreads, ((n + each - 1) / each + 31) & ~31);
  if (vec && threads == 32) return launch_chained(quantize_int8_kernel<T, true, true>, dim3((m + 7) / 8), dim3(32, 8), 0, s, in, ld, q, scales, m, k);
  return vec ? launch_chained(quantize_int8_kernel<T, true, false>, dim3(m), dim3(threads), 0, s, in, ld, q, scales, m, k)
             : launch_chained(quantize_int8_kernel<T, false, false>, dim3(m), dim3(threads), 0, s, in, ld, q, scales, m, k);
}

}  // namespace

int dense_sms() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  // tensor maps are encoded by the driver, which wants the device's context on this thread; one that has launched nothing yet has none
  thread_local int bound = -1;
  if (bound != dev) {
    if (cudaSetDevice(dev) != cudaSuccess) return 0;
    bound = dev;
  }
  return g_sms[dev].load();
}

EncodeFn dense_encoder() { return g_encode.load(); }

cudaError_t prepare_dense() {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (g_sms[dev].load() > 0) return cudaSuccess;
  if (g_encode.load() == nullptr) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess || fn == nullptr) return cudaErrorSymbolNotFound;
    g_encode.store(reinterpret_cast<EncodeFn>(fn));
  }
  e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess)
    e = for_each_pair_kernel([](auto kernel, bool, int, int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem); });
  if (e == cudaSuccess)
    e = for_each_few_kernel([](auto kernel, int, bool, int) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem); });
  for (int c = 2; c <= kFewMaxSplit && e == cudaSuccess; ++c) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c), cfg.blockDim = dim3(kFewThreads), cfg.dynamicSmemBytes = kFewSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, dense_few_kernel<true, false, kLinear>, &cfg);
    g_clusters[dev][c].store(n);
  }
  if (e == cudaSuccess) g_sms[dev].store(sms);
  return e;
}

// Few tokens: up to 192 where the weights are read along their rows (MN-major), else up to 160.  Few -> pairs, 5120 x 2304: 16-bit block, 128
// tokens 25.3 -> 28.7 us, 160 27.0 -> 28.7, 176 29.1 -> 28.7, 256 36.0 -> 29.0; 8-bit gated product, 160 11.2 -> 11.7, 176 12.1 -> 11.7.  Through the
// second product and to dx, 161 tokens 30.7 -> 37.1, 192 34.2 -> 37.3, 224 37.3 -> 37.4, 256 42.8 -> 37.7; all gradients (three launches, or two), 161
// 63.1 -> 76.2, 192 66.3 -> 76.2, 224 73.1 -> 74.8, 256 79.1 -> 75.2; of 8192 x 4096, 192 138 -> 185, 224 164 -> 162, 256 175 -> 164.  A small
// block would have its lines lower: 2048 x 1408, all gradients, 96 28.0 -> 29.6, 128 31.5 -> 30.0, 192 38.9 -> 30.2.
bool dense_few_tokens(const DenseProduct& p) { return !p.a.k_rows && p.m <= (p.b.k_rows ? kFewMaxTokens : kFewTokens); }

cudaError_t launch_dense(const DenseProduct* p, int parts, cudaStream_t s) {
  const int sms = dense_sms();
  if (sms == 0) return cudaErrorNotReady;
  const ChainScope chain(true);
  return parts == 1 && dense_few_tokens(*p) ? launch_few(*p, sms, s) : launch_pairs(p, parts, sms, s);
}

cudaError_t launch_quantize_int8(const void* x, int type, int64_t ld, int8_t* q, float* scales, int m, int k, cudaStream_t s) {
  if (m <= 0) return cudaSuccess;
  const ChainScope chain(true);
  return type == kDenseBf16 ? launch_quantize<__nv_bfloat16>(x, ld, q, scales, m, k, s) : launch_quantize<__half>(x, ld, q, scales, m, k, s);
}

}  // namespace mmoe
