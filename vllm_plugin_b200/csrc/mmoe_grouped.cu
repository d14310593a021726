// Products of a layer's experts for sm_100a (see mmoe_grouped.cuh).
#include <algorithm>

#include "mmoe_grouped_device.cuh"

namespace mmoe {

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Products on CTA pairs.  Weights are operand A (256 rows a tile, 128 in each CTA), an expert's rows operand B (up to 256 of them), so that what an
// expert without many rows costs goes by the number it has, in steps of 32.  A persistent pair takes tiles; which those are follows from
// `ends` alone, which every CTA reads for itself: nothing comes back to the host.
//
// Gate and up rows alternate by eights in a tile (one 5-D copy of the stored weights does that), so that tcgen05.ld.16x256b hands both values
// of a channel to the same thread.
//
// The sums stand with channels along the lanes and rows along the columns; stmatrix turns 8 x 8 blocks, and rows leave in 32 or 64 bytes.
//
// The gradient of the weights sums over an expert's rows.  Its last stage must not see the next expert's, whose values may be anything: the rows
// are copied through a 3-D view [rows][64 of them][columns] whose second extent ends the copy.  It starts as many rows early as are missing, and
// those are filled with zeros; the sum does not mind that they come first.
//
// What bounds it: the tensor cores, and in calls that last the power limit.  8 experts of 512 rows, gated 5120 -> 2 x 2304: 111 us (1.74 PFLOP/s; tensor
// cores 90 % busy, 435 MB of memory where 420 are the least) alone, 158 at 1.24 GHz of one call after another; a dense product of as many operations by the
// library 143.  46 experts with 23040 uneven rows, block 5120 -> 2304 -> 5120: 1.24 to 1.30 ms in bursts (1.25 to 1.31 PFLOP/s), 1.55 to 1.74 in calls that last, all
// their weights read beside it.  3840 rows of 7 experts with gradients: 710 to 720 us in bursts (1.1 PFLOP/s); through the second product 66 % and the gradients of the weights 68 to 73 % of the tensor cores' cycles,
// the rest goes into tiles that do not come out even and sums that leave (dw13 writes 378 MB).
// Where at most half of the pairs had a tile in the last turn, its tiles come in two halves of their columns (those of more than 128; fewer cost what the
// weights' bytes cost): 1021 rows of one expert, block with gradients 207 -> 184 us, 300 rows 122 -> 117, 3840 576 -> 567; not so the gradients of the
// weights, whose tiles are many.
//
// h, and in the backward pass dg and du, leave in the type of the operands: the next product multiplies them as such.  FP32 operands would be rounded as well (to
// TF32, eleven bits), at half the rate, with twice the bytes and weights that had to be widened.  The rounding takes a block's error against 64 bits from
// 0.0017 to 0.0024 of the result's norm in BF16 and from 0.00021 to 0.00029 in FP16; in FP16 an h past 65504 is an infinity.
//
// Tried: the widest tile chosen from 256, 224 ... 128 by the turns of the pairs, 186 us, but 48 experts with 6000 rows 593 -> 602.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kGroupCols = 256;                       // most rows of B per tile
constexpr int kGroupStageA = kGroupRows * 128;        // bytes
constexpr int kGroupStage = kGroupStageA + kGroupCols / 2 * 128;
constexpr int kGroupStages = 6;
constexpr int kGroupEpiWarps = 8;                     // two per TMEM lane quadrant, each with every other block of columns
constexpr int kGroupThreads = 32 * (2 + kGroupEpiWarps);
constexpr int kTurnBytes = 16 * 144;                  // a warp's 16 rows x 64 or 128 bytes, rows 80 or 144 bytes apart so that stmatrix meets no bank twice

struct GroupControl {
  uint64_t full[kGroupStages];    // leader only: every copy of the stage, in both CTAs, has landed
  uint64_t empty[kGroupStages];   // issuer -> producers of both CTAs
  uint64_t acc_full[2];           // issuer -> epilogues of both CTAs
  uint64_t acc_empty[2];          // leader only: epilogue warps of both CTAs -> issuer
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};

struct GroupedParams {
  CUtensorMap map_a;
  CUtensorMap map_b[4];           // boxes of 128, 64, 32 and 16 rows; kGroupedWeights: one
  const int32_t* ends;
  int32_t experts, rows;
  int32_t n, k;
  int32_t row_tiles;              // of an expert
  int32_t cols, col_tiles;        // kGroupedWeights
  int32_t k_stages;               // not kGroupedWeights
  uint32_t idesc;                 // without the columns
  DenseEpilogue epi;
  int32_t zero_behind;
  int32_t* status;
  int64_t timeout_ns;
};

constexpr int kGroupSmem = 227 * 1024;
constexpr int kGroupPlace = 1024;                                 // control block in front, the rest behind the stages
constexpr int kGroupStagesAt = kGroupPlace, kGroupPlanAt = kGroupStagesAt + kGroupStages * kGroupStage;
constexpr int kGroupTurnAt = kGroupPlanAt + (sizeof(GroupPlan) + 15) / 16 * 16;
static_assert(sizeof(GroupControl) <= kGroupPlace, "control block");
static_assert(kGroupTurnAt + kGroupEpiWarps * kTurnBytes + 1024 <= kGroupSmem, "shared memory of a CTA");

struct GroupTile {
  int expert, row0;               // first row of A, of the pair's tile
  int first, valid, cols;         // rows of x (first: of all); kGroupedWeights: columns
  int k_stages, k_first, k_rows;  // kGroupedWeights: the expert's rows
};

// The first `whole` tiles, then two parts of each of the others: halves of its columns, where it has more than 128, else all and none
template <int kKind>
__device__ __forceinline__ GroupTile tile_at(const GroupedParams& p, const GroupPlan* plan, int t, int whole) {
  GroupTile g;
  const int part = kKind != kGroupedWeights && t >= whole ? (t - whole) & 1 : -1;
  if (part >= 0) t = whole + (t - whole) / 2;
  if (kKind == kGroupedWeights) {
    const int each = p.row_tiles * p.col_tiles, in = t % each;
    g.expert = t / each;
    g.row0 = in / p.col_tiles * 2 * kGroupRows;
    g.first = in % p.col_tiles * p.cols;
    g.valid = min(p.k - g.first, p.cols), g.cols = p.cols;
    g.k_first = plan->start[g.expert], g.k_rows = plan->start[g.expert + 1] - g.k_first;
    g.k_stages = (g.k_rows + 63) / 64;
  } else {
    const int low = expert_of(*plan, p.experts, t);
    const int start = plan->start[low], count = plan->start[low + 1] - start, parts = (count + kGroupCols - 1) / kGroupCols;
    const int in = t - plan->tile[low], width = ((count + parts - 1) / parts + 31) & ~31, at = in % parts * width;
    g.expert = low;
    g.row0 = in / parts * (kKind == kGated ? kGroupRows : 2 * kGroupRows);
    g.first = start + at;
    g.valid = min(count - at, width), g.cols = (g.valid + 31) & ~31;
    g.k_stages = p.k_stages, g.k_first = g.k_rows = 0;
  }
  if (part >= 0) {
    const int cut = g.cols > 128 ? (g.cols / 2 + 31) & ~31 : g.cols;
    if (part == 0) g.valid = min(g.valid, cut), g.cols = cut;
    else g.first += cut, g.valid -= cut, g.cols -= cut;
  }
  return g;
}

// 32 columns of 16 lanes: v[4 g + 0 .. 3] = lane l / 4, columns 8 g + 2 (l % 4) and the next; then lane l / 4 + 8
__device__ __forceinline__ void tc_ld_fragments(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

template <typename T> __device__ __forceinline__ uint32_t pack_two(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_two<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_two<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool kTurned>
__device__ __forceinline__ void store_matrices(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  if (kTurned)
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
  else
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What a warp has to do with its part of a tile: 32 lanes (channels, or 16 of them with gate and up) by blocks of 32 columns
struct Share {
  uint8_t* turn;
  int lane;
  int channel0, channels;         // of the warp; where they end
};

// 16 rows of out (columns of the tile) x 32 channels.  v[h][g][r] as tc_ld_fragments gives them, h: lanes 16 on, for two g's
template <typename T>
__device__ __forceinline__ void put_rows(const Share& s, T* out, int64_t ld, int rows, const float (&v)[2][2][4]) {
  const int l = s.lane;
  __syncwarp();                                // the previous block has been read
#pragma unroll
  for (int g = 0; g < 2; ++g)
    store_matrices<true>(smem_u32(s.turn) + (8 * g + (l & 7)) * 80 + (l >> 3) * 16, pack_two<T>(v[0][g][0], v[0][g][1]),
                         pack_two<T>(v[0][g][2], v[0][g][3]), pack_two<T>(v[1][g][0], v[1][g][1]), pack_two<T>(v[1][g][2], v[1][g][3]));
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int row = 8 * g + (l >> 2), channel = s.channel0 + 8 * (l & 3);
    if (row < rows && channel < s.channels)
      *reinterpret_cast<uint4*>(out + row * ld + channel) = *reinterpret_cast<const uint4*>(s.turn + row * 80 + (l & 3) * 16);
  }
}
// the same of 16 channels: v[h][g][0, 1]
template <typename T>
__device__ __forceinline__ void put_half_rows(const Share& s, T* out, int64_t ld, int rows, const float (&v)[2][2][2]) {
  const int l = s.lane;
  __syncwarp();
  store_matrices<true>(smem_u32(s.turn) + (8 * (l >> 4) + (l & 7)) * 48 + ((l >> 3) & 1) * 16, pack_two<T>(v[0][0][0], v[0][0][1]),
                       pack_two<T>(v[1][0][0], v[1][0][1]), pack_two<T>(v[0][1][0], v[0][1][1]), pack_two<T>(v[1][1][0], v[1][1][1]));
  __syncwarp();
  const int row = l >> 1, channel = s.channel0 + 8 * (l & 1);
  if (row < rows && channel < s.channels)
    *reinterpret_cast<uint4*>(out + row * ld + channel) = *reinterpret_cast<const uint4*>(s.turn + row * 48 + (l & 1) * 16);
}
// 32 columns of a tile, of which `valid` exist, from row `first` of the output on.  v[h][g][r] with g = 0 .. 3
template <int kKind, typename T>
__device__ __forceinline__ void finish_columns_as(const DenseEpilogue& epi, const Share& s, int first, int valid, const float (&v)[2][4][4]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row0 = first + 16 * half, rows = valid - 16 * half;
    if (rows <= 0) break;
    if (kKind == kLinear) {
      float part[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) part[i >> 3][(i >> 2) & 1][i & 3] = v[i >> 3][2 * half + ((i >> 2) & 1)][i & 3];
      put_rows<T>(s, static_cast<T*>(epi.out) + (int64_t)row0 * epi.ld_out, epi.ld_out, rows, part);
    } else if (kKind == kGated) {
      float part[2][2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float gate = v[h][2 * half + g][r], up = v[h][2 * half + g][r + 2];
            part[h][g][r] = gated_value(gate, up, epi.clamp);
            if (epi.preact != nullptr) {
              const int row = 8 * g + 2 * (s.lane & 3) + r, channel = s.channel0 + 8 * h + (s.lane >> 2);
              if (row < rows && channel < s.channels) {
                float* keep = epi.preact + (int64_t)(row0 + row) * 2 * epi.inter + channel;
                keep[0] = gate, keep[epi.inter] = up;
              }
            }
          }
      put_half_rows<T>(s, static_cast<T*>(epi.out) + (int64_t)row0 * epi.ld_out, epi.ld_out, rows, part);
    } else {
      float dg[2][2][4], du[2][2][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int h = i >> 3, g = (i >> 2) & 1, r = i & 3, row = 8 * g + 2 * (s.lane & 3) + (r & 1), channel = s.channel0 + 16 * h + 8 * (r >> 1) + (s.lane >> 2);
        const bool there = row < rows && channel < s.channels;
        const float* keep = epi.preact + (int64_t)(row0 + row) * 2 * epi.inter + channel;
        dg[h][g][r] = there ? keep[0] : 0.f, du[h][g][r] = there ? keep[epi.inter] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int h = i >> 3, g = (i >> 2) & 1, r = i & 3;
        const float gate = dg[h][g][r], up = du[h][g][r];
        gated_grad(v[h][2 * half + g][r], gate, up, epi.clamp, dg[h][g][r], du[h][g][r]);
      }
      T* out = static_cast<T*>(epi.out) + (int64_t)row0 * epi.ld_out;
      put_rows<T>(s, out, epi.ld_out, rows, dg);
      put_rows<T>(s, out + epi.inter, epi.ld_out, rows, du);
    }
  }
}

// 64 columns x 32 rows of an expert's weights' gradient, which leave in 128 bytes of a row.  v[h][g][r] with g = 0 .. 7
template <typename T>
__device__ __forceinline__ void put_weights(const Share& s, T* out, int64_t ld, int column, int columns, const float (&v)[2][8][4]) {
  const int l = s.lane;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __syncwarp();
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int g = 0; g < 8; g += 4)
        store_matrices<false>(smem_u32(s.turn) + (8 * p + (l & 7)) * 144 + g * 16 + (l >> 3) * 16, pack_two<T>(v[h][g][2 * p], v[h][g][2 * p + 1]),
                              pack_two<T>(v[h][g + 1][2 * p], v[h][g + 1][2 * p + 1]), pack_two<T>(v[h][g + 2][2 * p], v[h][g + 2][2 * p + 1]),
                              pack_two<T>(v[h][g + 3][2 * p], v[h][g + 3][2 * p + 1]));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + (l >> 3), row = s.channel0 + 16 * h + r, at = column + 8 * (l & 7);
      if (row < s.channels && at < columns) *reinterpret_cast<uint4*>(out + row * ld + at) = *reinterpret_cast<const uint4*>(s.turn + r * 144 + (l & 7) * 16);
    }
  }
}
// ... of an expert without rows
template <typename T>
__device__ __forceinline__ void clear_weights(const Share& s, T* out, int64_t ld, int column, int columns) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = s.channel0 + 4 * i + (s.lane >> 3), at = column + 8 * (s.lane & 7);
    if (row < s.channels && at < columns) *reinterpret_cast<uint4*>(out + row * ld + at) = make_uint4(0, 0, 0, 0);
  }
}

template <int kKind>
__device__ __forceinline__ void finish_columns(const GroupedParams& p, const GroupTile& g, const Share& s, int column, const float (&v)[2][4][4]) {
  const DenseEpilogue& epi = p.epi;
  const int first = g.first + column, valid = g.valid - column;
  if (epi.out_type == kDenseBf16) finish_columns_as<kKind, __nv_bfloat16>(epi, s, first, valid, v);
  else finish_columns_as<kKind, __half>(epi, s, first, valid, v);
}

// kTurnedA, kTurnedB: the operand is staged with its rows along the 128 bytes (weights stored as [k, n]; both for the gradient of the weights)
template <int kKind, bool kTurnedA>
__global__ void __launch_bounds__(kGroupThreads, 1) grouped_pair_kernel(const __grid_constant__ GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in both CTAs
  GroupControl* ctl = reinterpret_cast<GroupControl*>(smem);
  uint8_t* stages = smem + kGroupStagesAt;
  GroupPlan* plan = reinterpret_cast<GroupPlan*>(smem + kGroupPlanAt);
  constexpr int kDepth = 64;                            // k's per stage
  constexpr bool kTurnedB = kKind == kGroupedWeights;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();
  if (threadIdx.x == 0) {
    prefetch_map(&p.map_a);
    for (int i = 0; i < (kTurnedB ? 1 : 4); ++i) prefetch_map(&p.map_b[i]);
    for (int i = 0; i < kGroupStages; ++i) {
      mbar_init(smem_u32(&ctl->full[i]), 1);
      mbar_init(smem_u32(&ctl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[i]), 2 * kGroupEpiWarps);
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
  int tiles = make_plan(plan, p.ends, p.experts, p.rows, kGroupCols, p.row_tiles, p.status);
  if (kKind == kGroupedWeights) tiles = p.experts * p.row_tiles * p.col_tiles;
  int whole = tiles;
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  const int step = gridDim.x / 2;
  if (kKind != kGroupedWeights && 2 * (tiles % step) <= step) whole = tiles / step * step, tiles += tiles - whole;        // the last turn in parts
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusGrouped, warp}, p.timeout_ns};
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
  if (p.zero_behind) {
    const int64_t row_bytes = p.epi.ld_out * 2, used = plan->start[p.experts];
    clear_bytes(static_cast<char*>(p.epi.out) + used * row_bytes, (p.rows - used) * row_bytes);
  }

  if (warp == 0) {
    // --------------------------------------------------------------------------------------------- producer
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t leader_full0 = map_to_cta(full0, 0), base = smem_u32(stages);
    bool ok = true;
    for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
      const GroupTile g = tile_at<kKind>(p, plan, t, whole);
      if (kKind != kGroupedWeights && g.valid <= 0) break;
      const int half = g.cols / 2;
      const uint32_t tx = 2 * (kGroupStageA + half * 128);
      const int a_row = g.row0 + static_cast<int>(cta) * (kKind == kGated ? kGroupRows / 2 : kGroupRows);
      const int b_row = g.first + static_cast<int>(cta) * half;
      for (int kb = 0; kb < g.k_stages; ++kb) {
        if (!waiter.wait_uniform(empty0 + 8 * stage, phase ^ 1u)) { ok = false; break; }
        const uint32_t bar = leader_full0 + 8 * stage, a = base + stage * kGroupStage, b = a + kGroupStageA;
        if (elect_one()) {
          if (cta == 0) mbar_expect_tx(full0 + 8 * stage, tx);
          if (kKind == kGroupedWeights) {
            const int at = kb * 64, missing = 64 - min(64, g.k_rows - at);
            pair_load_3d(a, &p.map_a, a_row, -missing, g.k_first + at, bar);
            pair_load_3d(a + 8192, &p.map_a, a_row + 64, -missing, g.k_first + at, bar);
            pair_load_3d(b, &p.map_b[0], b_row, -missing, g.k_first + at, bar);
            if (half > 64) pair_load_3d(b + 8192, &p.map_b[0], b_row + 64, -missing, g.k_first + at, bar);
          } else {
            if (kTurnedA) {
              pair_load_3d(a, &p.map_a, a_row, kb * kDepth, g.expert, bar);
              pair_load_3d(a + 8192, &p.map_a, a_row + 64, kb * kDepth, g.expert, bar);
            } else if (kKind == kGated) {
              pair_load_5d(a, &p.map_a, kb * kDepth, 0, 0, a_row / 8, g.expert, bar);
            } else {
              pair_load_3d(a, &p.map_a, kb * kDepth, a_row, g.expert, bar);
            }
            int done = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (half & (128 >> i)) {
                pair_load_2d(b + done * 128, &p.map_b[i], kb * kDepth, b_row + done, bar);
                done += 128 >> i;
              }
          }
        }
        __syncwarp();
        if (++stage == kGroupStages) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // --------------------------------------------------------------------------------------------- issuer
    if (cta == 0) {
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = true;
      const uint32_t lo0 = (smem_u32(stages) & 0x3FFFFu) >> 4;
      const uint64_t a_hi = operand_desc(kTurnedA, 8192), b_hi = operand_desc(kTurnedB, 8192);
      constexpr uint32_t kStepA = kTurnedA ? 2048 >> 4 : 2, kStepB = kTurnedB ? 2048 >> 4 : 2;
      for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
        const GroupTile g = tile_at<kKind>(p, plan, t, whole);
        if (kKind != kGroupedWeights && g.valid <= 0) break;
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(g.cols >> 3) << 17);
        if (!waiter.wait_uniform(smem_u32(&ctl->acc_empty[it & 1u]), ((it >> 1) & 1u) ^ 1u)) break;
        tc_fence_after();
        for (int kb = 0; kb < g.k_stages; ++kb) {
          if (!waiter.wait_uniform(full0 + 8 * stage, phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a = lo0 + stage * (kGroupStage >> 4), b = a + (kGroupStageA >> 4), d = tmem_base + (it & 1u) * kGroupCols;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) pair_product<false>(d, a_hi | (a + kStepA * k), b_hi | (b + kStepB * k), idesc, (kb | k) != 0 ? 1u : 0u);
            pair_commit(empty0 + 8 * stage);
          }
          __syncwarp();
          if (++stage == kGroupStages) { stage = 0; phase ^= 1u; }
        }
        if (ok && elect_one()) pair_commit(smem_u32(&ctl->acc_full[it & 1u]));
        __syncwarp();
        ++it;
      }
    }
  } else {
    // --------------------------------------------------------------------------------------------- epilogue
    const int quadrant = warp & 3;                    // of the TMEM lanes: the one this warp may read
    const int side = (warp - 2) >> 2;
    const uint32_t leader_empty = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    const uint32_t lanes = static_cast<uint32_t>(quadrant * 32) << 16;
    Share s;
    s.turn = smem + kGroupTurnAt + (warp - 2) * kTurnBytes, s.lane = lane, s.channels = p.n;
    uint32_t it = 0;
    for (int t = blockIdx.x / 2; t < tiles; t += step) {
      const GroupTile g = tile_at<kKind>(p, plan, t, whole);
      if (kKind != kGroupedWeights && g.valid <= 0) break;
      s.channel0 = g.row0 + (static_cast<int>(cta) * 4 + quadrant) * (kKind == kGated ? 16 : 32);
      const int blocks = (g.cols + 31) / 32;
      const auto release = [&](uint32_t acc) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(leader_empty + 8 * acc);
      };
      if (!waiter.wait_warp(smem_u32(&ctl->acc_full[it & 1u]), (it >> 1) & 1u, g.k_stages)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + (it & 1u) * kGroupCols + lanes;
      if constexpr (kKind == kGroupedWeights) {
        // two blocks at a time
        const int chunks = g.cols / 64;
        const int64_t at = (int64_t)g.expert * p.n * p.epi.ld_out;
        const auto each = [&](auto* out) {
          out += at;
#pragma unroll 1
          for (int chunk = side; chunk < chunks; chunk += 2) {
            if (g.k_stages == 0) {
              if (chunk + 2 >= chunks) release(it & 1u);
              clear_weights(s, out, p.epi.ld_out, g.first + 64 * chunk, p.k);
              continue;
            }
            float v[2][8][4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int b = 0; b < 2; ++b)
                tc_ld_fragments(d + 64 * chunk + 32 * b + (static_cast<uint32_t>(16 * h) << 16), reinterpret_cast<uint32_t*>(&v[h][4 * b][0]));
            tc_ld_wait();
            if (chunk + 2 >= chunks) release(it & 1u);
            put_weights(s, out, p.epi.ld_out, g.first + 64 * chunk, p.k, v);
          }
        };
        if (p.epi.out_type == kDenseBf16) each(static_cast<__nv_bfloat16*>(p.epi.out));
        else each(static_cast<__half*>(p.epi.out));
      } else {
        if (side >= blocks) release(it & 1u);
#pragma unroll 1
        for (int block = side; block < blocks; block += 2) {
          float v[2][4][4];
          uint32_t raw[32];
          tc_ld_fragments(d + 32 * block, raw);
          tc_ld_fragments(d + 32 * block + (16u << 16), raw + 16);
          tc_ld_wait();
          if (block + 2 >= blocks) release(it & 1u);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i >> 4][(i >> 2) & 3][i & 3] = __uint_as_float(raw[i]);
          finish_columns<kKind>(p, g, s, 32 * block, v);
        }
      }
      ++it;
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
// host
// ---------------------------------------------------------------------------------------------------------------------
// Weights [experts][n][k], boxes of a CTA's rows by 128 bytes of K; stored as [k][n] (k_rows): of 64 rows by 64 k's.  In three dimensions, so that a box
// ends with its expert.
bool encode_weights(CUtensorMap* map, const GroupedProduct& p) {
  const uint64_t n = p.n, k = p.k, e = p.experts;
  if (p.kind == kGated) {                      // eight gate rows, eight up rows, the next eight gate rows ...
    return encode_map(map, p.type, p.w, 5, {k, 8, 2, n / 8, e}, {2 * k, 2 * n * k, 16 * k, 4 * n * k}, {64, 8, 2, kGroupRows / 16, 1});
  }
  if (p.w_k_rows) return encode_map(map, p.type, p.w, 3, {n, k, e, 1, 1}, {2 * n, 2 * n * k, 0, 0}, {64, 64, 1, 1, 1});
  return encode_map(map, p.type, p.w, 3, {k, n, e, 1, 1}, {2 * k, 2 * n * k, 0, 0}, {64, kGroupRows, 1, 1, 1});
}

// Rows [rows][width], boxes of 128 bytes by `box` rows
bool encode_rows(CUtensorMap* map, const GroupedProduct& p, uint32_t box) {
  return encode_map(map, p.type, p.x, 2, {static_cast<uint64_t>(p.k), static_cast<uint64_t>(p.rows), 1, 1, 1}, {2 * static_cast<uint64_t>(p.x_ld), 0, 0, 0},
                    {64, box, 1, 1, 1});
}

// Rows as k's: [rows][64 of them][width], boxes of 64 columns by 64 rows from a given one on, where the 64 end
bool encode_summed(CUtensorMap* map, const GroupedProduct& p, const void* base, int64_t ld, uint64_t width) {
  const uint64_t pitch = 2 * static_cast<uint64_t>(ld);
  return encode_map(map, p.type, base, 3, {width, 64, static_cast<uint64_t>(p.rows), 1, 1}, {pitch, pitch, 0, 0}, {64, 64, 1, 1, 1});
}

template <typename F>
cudaError_t for_each_group_kernel(F f) {
  cudaError_t e = f(grouped_pair_kernel<kGated, false>, kGated, false);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<kLinear, false>, kLinear, false);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<kLinear, true>, kLinear, true);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<kGatedGrad, true>, kGatedGrad, true);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<kGroupedWeights, true>, kGroupedWeights, true);
  return e;
}

cudaError_t launch_group_pairs(const GroupedProduct& p, int sms, cudaStream_t s) {
  GroupedParams d = {};
  const bool weights = p.kind == kGroupedWeights, turned = weights || p.w_k_rows;
  d.ends = p.ends, d.experts = p.experts, d.rows = p.rows, d.n = p.n, d.k = p.k;
  const int rows = p.kind == kGated ? kGroupRows : 2 * kGroupRows;
  d.row_tiles = (p.n + rows - 1) / rows;
  d.k_stages = (p.k + 63) / 64;
  d.idesc = product_idesc(p.type, turned, weights, 2 * kGroupRows, 0);
  d.epi = p.epi;
  d.zero_behind = p.zero_behind && p.ends != nullptr;
  d.status = p.status;
  d.timeout_ns = (p.timeout_ms > 0 ? (int64_t)p.timeout_ms : 2000) * 1000000ll;
  bool ok = true;
  int64_t most;                                  // tiles
  if (weights) {
    d.cols = p.k > 128 ? 256 : 128;              // 64 columns of each CTA at least: a block of the copies
    d.col_tiles = (p.k + d.cols - 1) / d.cols;
    ok = encode_summed(&d.map_a, p, p.left, p.left_ld, p.n) && encode_summed(&d.map_b[0], p, p.x, p.x_ld, p.k);
    most = (int64_t)p.experts * d.row_tiles * d.col_tiles;
  } else {
    ok = encode_weights(&d.map_a, p);
    for (int i = 0; ok && i < 4; ++i) ok = encode_rows(&d.map_b[i], p, 128 >> i);
    most = ((int64_t)p.rows / kGroupCols + std::min(p.experts, p.rows)) * d.row_tiles;
  }
  if (!ok || most > INT32_MAX / 2) return cudaErrorInvalidValue;
  const int grid = 2 * static_cast<int>(std::min<int64_t>(sms / 2, 2 * most));       // every tile could come in two
  bool found = false;
  const cudaError_t e = for_each_group_kernel([&](auto kernel, int kind, bool k_turned) {
    if (kind != p.kind || k_turned != turned) return cudaSuccess;
    found = true;
    return launch_clustered(kernel, dim3(grid), dim3(kGroupThreads), kGroupSmem, 2, s, d);
  });
  return found ? e : cudaErrorInvalidValue;
}

}  // namespace

cudaError_t prepare_grouped() {
  return for_each_group_kernel([](auto kernel, int, bool) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmem); });
}

cudaError_t launch_grouped(const GroupedProduct& p, cudaStream_t s) {
  const int sms = dense_sms();
  if (sms == 0) return cudaErrorNotReady;
  const ChainScope chain(true);
  return grouped_few_rows(p, sms) ? launch_grouped_few(p, sms, s) : launch_group_pairs(p, sms, s);
}

}  // namespace mmoe
