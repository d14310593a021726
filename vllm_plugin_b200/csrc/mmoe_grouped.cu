// Products of a layer's experts for sm_100a (see mmoe_grouped.cuh).
#include <algorithm>

#include "mmoe_dense_device.cuh"
#include "mmoe_grouped.cuh"

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
// 8 bits: the tensor core sums one group of 128 k's; the epilogue warps multiply that by the two scales and add it to FP32 registers, beside the next
// group's products.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kGroupRows = 128;                       // rows of A per CTA
constexpr int kGroupCols = 256;                       // most rows of B per tile
constexpr int kGroupStageA = kGroupRows * 128;        // bytes
constexpr int kGroupStage = kGroupStageA + kGroupCols / 2 * 128;
constexpr int kGroupStages = 6;
constexpr int kGroupEpiWarps = 8;                     // two per TMEM lane quadrant, each with every other block of columns
constexpr int kGroupThreads = 32 * (2 + kGroupEpiWarps);
constexpr int kGroupScaleThreads = kGroupThreads + 32;          // 8 bits: one more warp, which fetches the scales
constexpr int kTurnBytes = 16 * 80;                   // a warp's 16 rows x 64 bytes, rows 80 bytes apart so that stmatrix meets no bank twice
constexpr int kScaleGroups = 4;                       // groups of k whose scales are fetched at a time
struct ScaleSlot {
  float x[kScaleGroups][kGroupCols];                  // by columns as the lanes want them (scale_place)
  float w[kScaleGroups][2];                           // gate (or only) and up rows
};

struct GroupControl {
  uint64_t full[kGroupStages];    // leader only: every copy of the stage, in both CTAs, has landed
  uint64_t empty[kGroupStages];   // issuer -> producers of both CTAs
  uint64_t acc_full[2];           // issuer -> epilogues of both CTAs
  uint64_t acc_empty[2];          // leader only: epilogue warps of both CTAs -> issuer
  uint64_t scale_full[2], scale_empty[2];
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};

// Where each expert's rows and tiles start
struct GroupPlan {
  int32_t start[kMaxExperts + 1];
  int32_t tile[kMaxExperts + 1];
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
  const float *x_scales, *w_scales;
  int32_t scale_groups, scale_blocks, scale_vectors;
  DenseEpilogue epi;
  int32_t zero_behind;
  int32_t* status;
  int64_t timeout_ns;
};

constexpr int kGroupSmem = 227 * 1024;
constexpr int kGroupPlace = 1024;                                 // control block in front, the rest behind the stages
constexpr int kGroupStagesAt = kGroupPlace, kGroupPlanAt = kGroupStagesAt + kGroupStages * kGroupStage;
constexpr int kGroupTurnAt = kGroupPlanAt + (sizeof(GroupPlan) + 15) / 16 * 16;
constexpr int kGroupScaleAt = kGroupTurnAt + kGroupEpiWarps * kTurnBytes;
static_assert(sizeof(GroupControl) <= kGroupPlace, "control block");
static_assert(kGroupScaleAt + 2 * sizeof(ScaleSlot) + 1024 <= kGroupSmem, "shared memory of a CTA");

struct GroupTile {
  int expert, row0;               // first row of A, of the pair's tile
  int first, valid, cols;         // rows of x (first: of all); kGroupedWeights: columns
  int k_stages, k_first, k_rows;  // kGroupedWeights: the expert's rows
};

// by all threads of a CTA; the number of tiles
template <int kKind>
__device__ __forceinline__ int make_plan(const GroupedParams& p, GroupPlan* plan) {
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) plan->start[e + 1] = p.ends != nullptr ? p.ends[e] : p.rows;
  if (threadIdx.x == 0) plan->start[0] = 0;
  __syncthreads();
  bool bad = threadIdx.x == 0 && plan->start[p.experts] > p.rows;
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) bad |= plan->start[e + 1] < plan->start[e];
  if (__syncthreads_or(bad)) {                 // nobody's rows then
    for (int e = threadIdx.x; e <= p.experts; e += blockDim.x) plan->start[e] = 0;
    if (threadIdx.x == 0 && blockIdx.x == 0) report_bad_index(p.status);
    __syncthreads();
  }
  if (kKind == kGroupedWeights) return p.experts * p.row_tiles * p.col_tiles;
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + threadIdx.x;
      int tiles = e < p.experts ? (plan->start[e + 1] - plan->start[e] + kGroupCols - 1) / kGroupCols * p.row_tiles : 0;
      const int own = tiles;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, tiles, d);
        if (threadIdx.x >= d) tiles += v;
      }
      if (e < p.experts) plan->tile[e] = sum + tiles - own;
      sum += __shfl_sync(0xffffffffu, tiles, 31);
    }
    if (threadIdx.x == 0) plan->tile[p.experts] = sum;
  }
  __syncthreads();
  return plan->tile[p.experts];
}

template <int kKind>
__device__ __forceinline__ GroupTile tile_at(const GroupedParams& p, const GroupPlan* plan, int t) {
  GroupTile g;
  if (kKind == kGroupedWeights) {
    const int each = p.row_tiles * p.col_tiles, in = t % each;
    g.expert = t / each;
    g.row0 = in / p.col_tiles * 2 * kGroupRows;
    g.first = in % p.col_tiles * p.cols;
    g.valid = min(p.k - g.first, p.cols), g.cols = p.cols;
    g.k_first = plan->start[g.expert], g.k_rows = plan->start[g.expert + 1] - g.k_first;
    g.k_stages = (g.k_rows + 63) / 64;
    return g;
  }
  int low = 0, high = p.experts;               // tile[low] <= t < tile[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (plan->tile[mid] <= t) low = mid;
    else high = mid;
  }
  const int start = plan->start[low], count = plan->start[low + 1] - start, parts = (count + kGroupCols - 1) / kGroupCols;
  const int in = t - plan->tile[low], width = ((count + parts - 1) / parts + 31) & ~31, at = in % parts * width;
  g.expert = low;
  g.row0 = in / parts * (kKind == kGated ? kGroupRows : 2 * kGroupRows);
  g.first = start + at;
  g.valid = min(count - at, width), g.cols = (g.valid + 31) & ~31;
  g.k_stages = p.k_stages, g.k_first = g.k_rows = 0;
  return g;
}

// zeros from p on, by all threads of the grid
__device__ __forceinline__ void clear_bytes(char* p, int64_t bytes) {
  const int64_t thread = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15)), body = (bytes - head) / 16;
  for (int64_t i = thread; i < head; i += threads) p[i] = 0;
  for (int64_t i = thread; i < body; i += threads) reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = head + body * 16 + thread; i < bytes; i += threads) p[i] = 0;
}

__device__ __forceinline__ void pair_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}

template <bool kFp8>
__device__ __forceinline__ void group_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kFp8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    pair_product<false>(d, a, b, idesc, accumulate);
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
constexpr int kScalePlaceStride = 8;
// where a column's scale lies among its block of 32: the eight that lane l % 4 wants are neighbours
__device__ __forceinline__ int scale_place(int c) { return (c & ~31) + ((c & 7) >> 1) * kScalePlaceStride + ((c >> 3) & 3) * 2 + (c & 1); }

__device__ __forceinline__ uint64_t two_floats(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 both_floats(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
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
  if ((s.channels & 7) != 0) {                 // rows that start anywhere
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 8 * g + 2 * (l & 3) + (r & 1), channel = s.channel0 + 16 * h + 8 * (r >> 1) + (l >> 2);
          if (row < rows && channel < s.channels) out[row * ld + channel] = from_float<T>(v[h][g][r]);
        }
    return;
  }
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
template <>
__device__ __forceinline__ void put_rows<float>(const Share& s, float* out, int64_t ld, int rows, const float (&v)[2][2][4]) {
  // eight lanes write eight neighbours
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 8 * g + 2 * (s.lane & 3) + (r & 1), channel = s.channel0 + 16 * h + 8 * (r >> 1) + (s.lane >> 2);
        if (row < rows && channel < s.channels) out[row * ld + channel] = v[h][g][r];
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
template <>
__device__ __forceinline__ void put_half_rows<float>(const Share& s, float* out, int64_t ld, int rows, const float (&v)[2][2][2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 8 * g + 2 * (s.lane & 3) + r, channel = s.channel0 + 8 * h + (s.lane >> 2);
        if (row < rows && channel < s.channels) out[row * ld + channel] = v[h][g][r];
      }
}

// 32 columns of a tile, of which `valid` exist, from row `first` of the output on.  v[h][g][r] with g = 0 .. 3
template <bool kFp8, int kKind, typename T>
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
            part[h][g][r] = kFp8 && sizeof(T) == 4 ? gated_value_fp32(gate, up, epi.clamp) : gated_value(gate, up, epi.clamp);
            if (!kFp8 && epi.preact != nullptr) {
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

// 32 columns x 32 rows of an expert's weights' gradient
template <typename T>
__device__ __forceinline__ void put_weights(const Share& s, T* out, int64_t ld, int column, int columns, const float (&v)[2][4][4]) {
  const int l = s.lane;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    __syncwarp();
#pragma unroll
    for (int p = 0; p < 2; ++p)
      store_matrices<false>(smem_u32(s.turn) + (8 * p + (l & 7)) * 80 + (l >> 3) * 16, pack_two<T>(v[h][0][2 * p], v[h][0][2 * p + 1]),
                            pack_two<T>(v[h][1][2 * p], v[h][1][2 * p + 1]), pack_two<T>(v[h][2][2 * p], v[h][2][2 * p + 1]),
                            pack_two<T>(v[h][3][2 * p], v[h][3][2 * p + 1]));
    __syncwarp();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = s.channel0 + 16 * h + 8 * p + (l >> 2), at = column + 8 * (l & 3);
      if (row < s.channels && at < columns)
        *reinterpret_cast<uint4*>(out + row * ld + at) = *reinterpret_cast<const uint4*>(s.turn + (8 * p + (l >> 2)) * 80 + (l & 3) * 16);
    }
  }
}

template <bool kFp8, int kKind>
__device__ __forceinline__ void finish_columns(const GroupedParams& p, const GroupTile& g, const Share& s, int column, const float (&v)[2][4][4]) {
  const DenseEpilogue& epi = p.epi;
  if (kKind == kGroupedWeights) {
    const int64_t at = (int64_t)g.expert * p.n * epi.ld_out;
    if (epi.out_type == kDenseBf16) put_weights(s, static_cast<__nv_bfloat16*>(epi.out) + at, epi.ld_out, g.first + column, p.k, v);
    else put_weights(s, static_cast<__half*>(epi.out) + at, epi.ld_out, g.first + column, p.k, v);
    return;
  }
  const int first = g.first + column, valid = g.valid - column;
  if constexpr (kKind != kGroupedWeights) {
    if (epi.out_type == kDenseBf16) finish_columns_as<kFp8, kKind, __nv_bfloat16>(epi, s, first, valid, v);
    else if (epi.out_type == kDenseFp16) finish_columns_as<kFp8, kKind, __half>(epi, s, first, valid, v);
    else if constexpr (kFp8) finish_columns_as<kFp8, kKind, float>(epi, s, first, valid, v);
  }
}

// kTurnedA, kTurnedB: the operand is staged with its rows along the 128 bytes (weights stored as [k, n]; both for the gradient of the weights)
template <bool kFp8, int kKind, bool kTurnedA>
__global__ void __launch_bounds__(kFp8 ? kGroupScaleThreads : kGroupThreads, 1) grouped_pair_kernel(const __grid_constant__ GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in both CTAs
  GroupControl* ctl = reinterpret_cast<GroupControl*>(smem);
  uint8_t* stages = smem + kGroupStagesAt;
  GroupPlan* plan = reinterpret_cast<GroupPlan*>(smem + kGroupPlanAt);
  ScaleSlot* slots = reinterpret_cast<ScaleSlot*>(smem + kGroupScaleAt);
  constexpr int kDepth = kFp8 ? 128 : 64;               // k's per stage
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
      mbar_init(smem_u32(&ctl->scale_full[i]), 1);
      mbar_init(smem_u32(&ctl->scale_empty[i]), kGroupEpiWarps);
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
  const int tiles = make_plan<kKind>(p, plan);
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  const int step = gridDim.x / 2;
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusGrouped, warp}, p.timeout_ns};
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
  if (p.zero_behind) {
    const int64_t row_bytes = p.epi.ld_out * (p.epi.out_type == kDenseFp32 ? 4 : 2), used = plan->start[p.experts];
    clear_bytes(static_cast<char*>(p.epi.out) + used * row_bytes, (p.rows - used) * row_bytes);
  }

  if (warp == 0) {
    // --------------------------------------------------------------------------------------------- producer
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t leader_full0 = map_to_cta(full0, 0), base = smem_u32(stages);
    bool ok = true;
    for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
      const GroupTile g = tile_at<kKind>(p, plan, t);
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
        const GroupTile g = tile_at<kKind>(p, plan, t);
        const uint32_t idesc = p.idesc | (static_cast<uint32_t>(g.cols >> 3) << 17);
        const auto open = [&] {              // an accumulator
          if (!waiter.wait_uniform(smem_u32(&ctl->acc_empty[it & 1u]), ((it >> 1) & 1u) ^ 1u)) return false;
          tc_fence_after();
          return true;
        };
        const auto close = [&] {
          if (elect_one()) pair_commit(smem_u32(&ctl->acc_full[it & 1u]));
          __syncwarp();
          ++it;
        };
        if (!kFp8 && !open()) break;
        for (int kb = 0; kb < g.k_stages; ++kb) {
          if (kFp8 && !open()) { ok = false; break; }
          if (!waiter.wait_uniform(full0 + 8 * stage, phase)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a = lo0 + stage * (kGroupStage >> 4), b = a + (kGroupStageA >> 4), d = tmem_base + (it & 1u) * kGroupCols;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              group_product<kFp8>(d, a_hi | (a + kStepA * k), b_hi | (b + kStepB * k), idesc, ((kFp8 ? 0 : kb) | k) != 0 ? 1u : 0u);
            pair_commit(empty0 + 8 * stage);
          }
          __syncwarp();
          if (kFp8) close();
          if (++stage == kGroupStages) { stage = 0; phase ^= 1u; }
        }
        if (!kFp8 && ok) close();
      }
    }
  } else if (kFp8 && warp == 2 + kGroupEpiWarps) {
    // --------------------------------------------------------------------------------------------- scales
    uint32_t it = 0;
    bool ok = true;
    for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
      const GroupTile g = tile_at<kKind>(p, plan, t);
      const int block = (g.row0 + static_cast<int>(cta) * (kKind == kGated ? kGroupRows / 2 : kGroupRows)) / kScaleBlock;
      const int blocks = kKind == kGated ? p.scale_blocks / 2 : p.scale_blocks;
      const float* w = p.w_scales + ((int64_t)g.expert * p.scale_blocks + min(block, blocks - 1)) * p.scale_groups;
      for (int kb = 0; kb < g.k_stages; kb += kScaleGroups, ++it) {
        ScaleSlot* slot = &slots[it & 1u];
        const int groups = min(kScaleGroups, g.k_stages - kb);
        // on their way while the slot is still in use
        float v[kGroupCols / 32][kScaleGroups], ws = 0.f;
#pragma unroll
        for (int i = 0; i < kGroupCols / 32; ++i) {
          const int c = 32 * i + lane;
          const float* src = p.x_scales + (int64_t)(g.first + c) * p.scale_groups + kb;
          if (p.scale_vectors && groups == kScaleGroups) {
            const float4 f = c < g.valid ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
          } else {
#pragma unroll
            for (int j = 0; j < kScaleGroups; ++j) v[i][j] = c < g.valid && j < groups ? src[j] : 0.f;
          }
        }
        if (lane < 2 * kScaleGroups && (lane >> 1) < groups && ((lane & 1) == 0 || kKind == kGated))
          ws = w[(lane & 1) * (int64_t)blocks * p.scale_groups + kb + (lane >> 1)];
        if (!waiter.wait_warp(smem_u32(&ctl->scale_empty[it & 1u]), ((it >> 1) & 1u) ^ 1u, kScaleGroups)) { ok = false; break; }
#pragma unroll
        for (int i = 0; i < kGroupCols / 32; ++i) {
#pragma unroll
          for (int j = 0; j < kScaleGroups; ++j) slot->x[j][scale_place(32 * i + lane)] = v[i][j];
        }
        if (lane < 2 * kScaleGroups) slot->w[lane >> 1][lane & 1] = ws;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->scale_full[it & 1u]));
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
    uint32_t it = 0, slot_it = 0;
    bool ok = true;
    for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
      const GroupTile g = tile_at<kKind>(p, plan, t);
      s.channel0 = g.row0 + (static_cast<int>(cta) * 4 + quadrant) * (kKind == kGated ? 16 : 32);
      const int blocks = (g.cols + 31) / 32;
      const auto release = [&](uint32_t acc) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_pair(leader_empty + 8 * acc);
      };
      if constexpr (kFp8) {
        uint64_t sum[4][2][4][2] = {};       // by [block][lanes 16 on][group of 8 columns][lane + 8]
        for (int kb = 0; kb < g.k_stages; ++kb, ++it) {
          const int in = kb % kScaleGroups;
          if (in == 0 && !waiter.wait_warp(smem_u32(&ctl->scale_full[slot_it & 1u]), (slot_it >> 1) & 1u, kScaleGroups)) { ok = false; break; }
          const ScaleSlot& slot = slots[slot_it & 1u];
          const uint64_t w0 = two_floats(slot.w[in][0], slot.w[in][0]), w1 = two_floats(slot.w[in][1], slot.w[in][1]);
          if (!waiter.wait_warp(smem_u32(&ctl->acc_full[it & 1u]), (it >> 1) & 1u, 1)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem_base + (it & 1u) * kGroupCols + lanes;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int block = 2 * b + side;
            if (block < blocks) {
              uint32_t v[32];
              tc_ld_fragments(d + 32 * block, v);
              tc_ld_fragments(d + 32 * block + (16u << 16), v + 16);
              const ulonglong2* from = reinterpret_cast<const ulonglong2*>(&slot.x[in][32 * block + (lane & 3) * kScalePlaceStride]);
              const ulonglong2 s01 = from[0], s23 = from[1];
              const uint64_t sx[4] = {s01.x, s01.y, s23.x, s23.y};
              tc_ld_wait();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint64_t f0 = mul_two(sx[i], w0), f1 = kKind == kGated ? mul_two(sx[i], w1) : f0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t* q = v + 16 * h + 4 * i;
                  sum[b][h][i][0] = fma_two(two_floats(__uint_as_float(q[0]), __uint_as_float(q[1])), f0, sum[b][h][i][0]);
                  sum[b][h][i][1] = fma_two(two_floats(__uint_as_float(q[2]), __uint_as_float(q[3])), f1, sum[b][h][i][1]);
                }
              }
            }
          }
          release(it & 1u);
          if (in == kScaleGroups - 1 || kb == g.k_stages - 1) {
            if (lane == 0) mbar_arrive(smem_u32(&ctl->scale_empty[slot_it & 1u]));
            ++slot_it;
          }
        }
        if (ok) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int block = 2 * b + side;
            if (block < blocks) {
              float v[2][4][4];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 f = both_floats(sum[b][i >> 3][(i >> 1) & 3][i & 1]);
                v[i >> 3][(i >> 1) & 3][2 * (i & 1)] = f.x, v[i >> 3][(i >> 1) & 3][2 * (i & 1) + 1] = f.y;
              }
              finish_columns<kFp8, kKind>(p, g, s, 32 * block, v);
            }
          }
        }
      } else {
        if (!waiter.wait_warp(smem_u32(&ctl->acc_full[it & 1u]), (it >> 1) & 1u, g.k_stages)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + (it & 1u) * kGroupCols + lanes;
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
          for (int i = 0; i < 32; ++i) v[i >> 4][(i >> 2) & 3][i & 3] = kKind == kGroupedWeights && g.k_stages == 0 ? 0.f : __uint_as_float(raw[i]);
          finish_columns<kFp8, kKind>(p, g, s, 32 * block, v);
        }
        ++it;
      }
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
bool encode_map(CUtensorMap* map, int type, const void* base, int rank, const uint64_t (&dims)[5], const uint64_t (&strides)[4], const uint32_t (&box)[5]) {
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType t = type == kGroupedE4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == kDenseBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t d[5], st[4];
  cuuint32_t b[5];
  std::copy(dims, dims + 5, d), std::copy(strides, strides + 4, st), std::copy(box, box + 5, b);
  return dense_encoder()(map, t, rank, const_cast<void*>(base), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Weights [experts][n][k], boxes of `box` rows by 128 bytes of K; stored as [k][n] (k_rows): of 64 rows by 64 k's.  In three dimensions, so that a box
// ends with its expert.
bool encode_weights(CUtensorMap* map, const GroupedProduct& p, uint32_t box) {
  const uint64_t size = p.type == kGroupedE4m3 ? 1 : 2, n = p.n, k = p.k, e = p.experts;
  if (p.kind == kGated) {                      // eight gate rows, eight up rows, the next eight gate rows ...
    return encode_map(map, p.type, p.w, 5, {k, 8, 2, n / 8, e}, {k * size, n * k * size, 8 * k * size, 2 * n * k * size},
                      {static_cast<uint32_t>(128 / size), 8, 2, box / 16, 1});
  }
  if (p.w_k_rows) return encode_map(map, p.type, p.w, 3, {n, k, e, 1, 1}, {n * size, n * k * size, 0, 0}, {64, 64, 1, 1, 1});
  return encode_map(map, p.type, p.w, 3, {k, n, e, 1, 1}, {k * size, n * k * size, 0, 0}, {static_cast<uint32_t>(128 / size), box, 1, 1, 1});
}

// Rows [rows][width], boxes of 128 bytes by `box` rows
bool encode_rows(CUtensorMap* map, const GroupedProduct& p, uint32_t box) {
  const uint64_t size = p.type == kGroupedE4m3 ? 1 : 2;
  return encode_map(map, p.type, p.x, 2, {static_cast<uint64_t>(p.k), static_cast<uint64_t>(p.rows), 1, 1, 1}, {p.x_ld * size, 0, 0, 0},
                    {static_cast<uint32_t>(128 / size), box, 1, 1, 1});
}

// Rows as k's: [rows][64 of them][width], boxes of 64 columns by 64 rows from a given one on, where the 64 end
bool encode_summed(CUtensorMap* map, const GroupedProduct& p, const void* base, int64_t ld, uint64_t width) {
  const uint64_t pitch = 2 * static_cast<uint64_t>(ld);
  return encode_map(map, p.type, base, 3, {width, 64, static_cast<uint64_t>(p.rows), 1, 1}, {pitch, pitch, 0, 0}, {64, 64, 1, 1, 1});
}

template <typename F>
cudaError_t for_each_group_kernel(F f) {
  cudaError_t e = f(grouped_pair_kernel<false, kGated, false>, false, kGated, false);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<false, kLinear, false>, false, kLinear, false);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<false, kLinear, true>, false, kLinear, true);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<false, kGatedGrad, true>, false, kGatedGrad, true);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<false, kGroupedWeights, true>, false, kGroupedWeights, true);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<true, kGated, false>, true, kGated, false);
  if (e == cudaSuccess) e = f(grouped_pair_kernel<true, kLinear, false>, true, kLinear, false);
  return e;
}

cudaError_t launch_group_pairs(const GroupedProduct& p, int sms, cudaStream_t s) {
  GroupedParams d = {};
  const bool fp8 = p.type == kGroupedE4m3, weights = p.kind == kGroupedWeights, turned = weights || p.w_k_rows;
  d.ends = p.ends, d.experts = p.experts, d.rows = p.rows, d.n = p.n, d.k = p.k;
  const int rows = p.kind == kGated ? kGroupRows : 2 * kGroupRows, depth = fp8 ? 128 : 64;
  d.row_tiles = (p.n + rows - 1) / rows;
  d.k_stages = (p.k + depth - 1) / depth;
  d.idesc = product_idesc(fp8 ? kDenseFp16 : p.type, turned, weights, 2 * kGroupRows, 0);      // format 0: FP16, or in 8 bits E4M3
  d.x_scales = p.x_scales, d.w_scales = p.w_scales;
  d.scale_groups = (p.k + kScaleBlock - 1) / kScaleBlock;
  d.scale_blocks = (p.n + kScaleBlock - 1) / kScaleBlock * (p.kind == kGated ? 2 : 1);
  d.scale_vectors = d.scale_groups % kScaleGroups == 0 && reinterpret_cast<uintptr_t>(p.x_scales) % 16 == 0;
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
    ok = encode_weights(&d.map_a, p, kGroupRows);
    for (int i = 0; ok && i < 4; ++i) ok = encode_rows(&d.map_b[i], p, 128 >> i);
    most = ((int64_t)p.rows / kGroupCols + std::min(p.experts, p.rows)) * d.row_tiles;
  }
  if (!ok || most > INT32_MAX / 2) return cudaErrorInvalidValue;
  const int grid = 2 * static_cast<int>(std::min<int64_t>(sms / 2, most));
  bool found = false;
  const cudaError_t e = for_each_group_kernel([&](auto kernel, bool k_fp8, int kind, bool k_turned) {
    if (k_fp8 != fp8 || kind != p.kind || k_turned != turned) return cudaSuccess;
    found = true;
    return launch_clustered(kernel, dim3(grid), dim3(fp8 ? kGroupScaleThreads : kGroupThreads), kGroupSmem, 2, s, d);
  });
  return found ? e : cudaErrorInvalidValue;
}

// ---------------------------------------------------------------------------------------------------------------------
// Quantiser: s = max|x| / 448 for each 128 values of a row, q = x / s rounded to the nearest E4M3 value, ties to even.
// Sixteen lanes have a group, eight values each, which stay in registers between the maximum and the quotients.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 256, kQuantLanes = 16;

// x / s in E4M3, exactly, two values.  The product with the reciprocal is within 2^-22 of the quotient, which matters next to a border between two E4M3
// values alone: there the 20 bits that E4M3 drops are near their middle (of a number below 2^-6, where the steps are those of [2^-6, 2^-5): when 2^-6 is
// added).  Then the quotient is taken with its last bit set where it is not exact, which rounds as the exact one does.
__device__ __forceinline__ bool near_border(float q) {
  const float a = fabsf(q), z = a < 0x1p-6f ? a + 0x1p-6f : a;
  return ((__float_as_uint(z) - 0x80000u + 8u) & 0xfffffu) < 16u;
}
__device__ __forceinline__ float odd_quotient(float x, float s) {
  const float q = __fdiv_rn(x, s), rest = fmaf(-q, s, x);
  uint32_t bits = __float_as_uint(q);
  if (rest != 0.f) {
    if ((rest < 0.f) != (q < 0.f)) --bits;       // towards zero ...
    bits |= 1u;                                  // ... and marked
  }
  return __uint_as_float(bits);
}
__device__ __forceinline__ uint32_t two_e4m3(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// kVec: eight neighbouring values in one load; else (widths, strides or places that do not allow it) every sixteenth
template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) quantize_fp8_kernel(const T* x, int64_t ld, uint8_t* q, float* scales, uint32_t total, uint32_t groups, int k) {
  chain_wait();
  chain_release();
  const uint64_t index = (uint64_t)blockIdx.x * (kQuantThreads / kQuantLanes) + threadIdx.x / kQuantLanes;
  const bool there = index < total;            // sixteen lanes alike
  const uint32_t row = static_cast<uint32_t>(index) / groups, group = static_cast<uint32_t>(index) - row * groups;
  const int lane = threadIdx.x % kQuantLanes, first = static_cast<int>(group) * kScaleBlock, count = there ? min(kScaleBlock, k - first) : 0;
  const T* in = x + row * ld + first;
  float v[8];
  if constexpr (kVec) {
    struct alignas(16) Vec { T v[8]; };
    Vec f = {};
    if (8 * lane < count) f = *reinterpret_cast<const Vec*>(in + 8 * lane);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(f.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = lane + 16 * j < count ? static_cast<float>(in[lane + 16 * j]) : 0.f;
  }
  // magnitudes as bits: NaN is above infinity there, so neither is lost
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
  for (int d = kQuantLanes / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  const bool finite = top < 0x7f800000u;
  float s = !finite ? __uint_as_float(0x7fffffffu) : top == 0 ? 1.f : __fdiv_rn(__uint_as_float(top), 448.f);
  if (there && lane == 0) scales[(int64_t)row * groups + group] = s;
  if (s < 0x1p-60f) {                          // remainders of quotients by so small a scale would be no numbers
    s *= 0x1p80f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= 0x1p80f;
  }
  const float inv = __fdiv_rn(1.f, s);
  float r[8];
  bool near = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    r[j] = finite ? v[j] * inv : 0.f;
    near |= near_border(r[j]);
  }
  if (near) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = odd_quotient(v[j], s);
  }
  uint8_t* out = q + (int64_t)row * k + first;
  const uint32_t b[4] = {two_e4m3(r[0], r[1]), two_e4m3(r[2], r[3]), two_e4m3(r[4], r[5]), two_e4m3(r[6], r[7])};
  if constexpr (kVec) {
    if (8 * lane < count) *reinterpret_cast<uint2*>(out + 8 * lane) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 16 * j < count) out[lane + 16 * j] = static_cast<uint8_t>(b[j / 2] >> (j & 1) * 8);
  }
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t ld, uint8_t* q, float* scales, int m, int k, cudaStream_t s) {
  const T* in = static_cast<const T*>(x);
  const bool vec = k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const uint32_t groups = (static_cast<uint32_t>(k) + kScaleBlock - 1) / kScaleBlock;
  const uint64_t total = (uint64_t)m * groups, blocks = (total + kQuantThreads / kQuantLanes - 1) / (kQuantThreads / kQuantLanes);
  if (total > UINT32_MAX || blocks > INT32_MAX) return cudaErrorInvalidValue;
  const uint32_t n = static_cast<uint32_t>(total);
  return vec ? launch_chained(quantize_fp8_kernel<T, true>, dim3(static_cast<uint32_t>(blocks)), dim3(kQuantThreads), 0, s, in, ld, q, scales, n, groups, k)
             : launch_chained(quantize_fp8_kernel<T, false>, dim3(static_cast<uint32_t>(blocks)), dim3(kQuantThreads), 0, s, in, ld, q, scales, n, groups, k);
}

}  // namespace

cudaError_t prepare_grouped() {
  return for_each_group_kernel([](auto kernel, bool, int, bool) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmem); });
}

cudaError_t launch_grouped(const GroupedProduct& p, cudaStream_t s) {
  const int sms = dense_sms();
  if (sms == 0) return cudaErrorNotReady;
  const ChainScope chain(true);
  return launch_group_pairs(p, sms, s);
}

cudaError_t launch_quantize_fp8(const void* x, int type, int64_t ld, uint8_t* q, float* scales, int m, int k, cudaStream_t s) {
  if (m <= 0) return cudaSuccess;
  const ChainScope chain(true);
  return type == kDenseBf16 ? launch_quantize<__nv_bfloat16>(x, ld, q, scales, m, k, s) : launch_quantize<__half>(x, ld, q, scales, m, k, s);
}

}  // namespace mmoe
