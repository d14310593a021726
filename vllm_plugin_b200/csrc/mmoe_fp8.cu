// Products in 8-bit floating point with block scales for sm_100a (see mmoe_grouped.cuh), and the quantiser in front of them.
#include <algorithm>
#include <type_traits>

#include "mmoe_grouped_device.cuh"

namespace mmoe {

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Products on CTA pairs: out[t, n] = sum over groups kb of 128 k's of (sum_k x[t, k] w[n, k]) sx[t, kb] sw[n / 128, kb].
// Rows are operand A (256 a tile, 128 in each CTA), weights operand B (256 a tile; gated: half of them gate rows, which the leader stages, the up rows its
// peer).  The tensor core sums one group into two accumulators of 128 columns, one after the other, of four; the epilogue warps multiply them by the two scales
// and add them to FP32 registers, beside the next products.  Four warps have one accumulator of a group, four the other.  A thread has one row of the tile,
// so that its scale is one number a group; weights' scales are one for every 32 columns.  (Weights along the lanes instead: a scale for every column and
// thread, 109 us where this form began with 55.)  Columns come by sixteens beside the multiplications of the sixteen before, the next group's first ones too: 54.5
// -> 50.7 us of a linear and 96 -> 90 of a gated product below.  One warp brings the scales, word by word and up to three batches ahead.
//
// Where at most half of the pairs had a tile in the last turn, its tiles come in two halves of their columns: one accumulator a group, which all
// warps share.  50.7 -> 49.2 us (300 tiles for 74 pairs); 1021 rows, 5120 -> 5003 (80) 52.8 -> 46.1.
//
// What bounds it: the power limit, in calls that last.  3840 rows, 2304 -> 5120 49 us in bursts and 54.5 repeated (1.66-1.85 PFLOP/s), gated 5120 -> 2 x 2304 84
// and 98 us (1.85-2.16).  With nothing done by the epilogue warps, 38.5 and 70 us in bursts and 46 and 83 repeated (at 1.55 GHz): that is what
// products and copies alone would take.  Multiplications take another 6 and 9, writing the results, which the next tile's sums wait for, 6 and 6.
// Tried, linear and gated (49 and then 90): all warps with 64 columns of each accumulator 56, 102; one accumulator of 256 columns a group 51, 92; 24 columns at
// a time 51.6, 90.9, and 32, for which registers are short, 53.8, 94; packed pairs (fma.rn.f32x2) 50, 89 and 55.3, 103 repeated; waits of the issuing warp
// that put it to sleep 53, 96; one thread that issues 66, 128.  Before columns came by sixteens (54.5, 93): sixteen epilogue warps with 64 columns each 63, 97;
// tiles of 192 columns 88, 160; eight groups' scales by the epilogue warps themselves 60, 102.  When these were 49 and 84: results by one bulk copy a row 55, 86; by a
// warp of their own, with four stages instead of five, 50, 87.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kFp8Unit = 128;                         // columns of an accumulator
constexpr int kFp8Units = kTmemCols / kFp8Unit;
constexpr int kFp8Cols = 2 * kFp8Unit;                // rows of B per tile
constexpr int kFp8StageA = kGroupRows * 128;          // bytes
constexpr int kFp8StageHalf = kFp8Unit / 2 * 128;     // of B, for one of the tile's accumulators
constexpr int kFp8Stage = kFp8StageA + 2 * kFp8StageHalf;
constexpr int kFp8Stages = 5;
constexpr int kFp8EpiWarps = 8;                       // two per TMEM lane quadrant, each with half of an accumulator's columns
constexpr int kFp8Threads = 32 * (4 + kFp8EpiWarps);   // epilogue warps first, producer, issuer, one that fetches scales, one that only hands back registers
constexpr int kFp8Registers = 208, kFp8FewRegisters = 88;
static_assert(kFp8EpiWarps * 32 * kFp8Registers + 128 * kFp8FewRegisters <= kFp8Threads * 168, "registers that the block was launched with");
constexpr int kFp8Batch = 8;                          // groups of k whose scales are fetched at a time
constexpr int kFp8Turn = 32 * 144;                    // a warp's 32 rows x 128 bytes on their way from lanes to rows
constexpr int kFp8ScaleSlots = 4;
// scales of a batch
struct Fp8Scales {
  float x[kFp8Batch][kGroupRows + 4];                 // of the CTA's rows; padded so that four rows x eight groups are written to 32 banks
  float w[kFp8Batch][8];                              // of the blocks of 32 columns, by warp side
};

struct Fp8Control {
  uint64_t full[kFp8Stages];         // leader only: every copy of the stage, in both CTAs, has landed
  uint64_t empty[kFp8Stages];        // issuer -> producers of both CTAs
  uint64_t acc_full[kFp8Units];           // issuer -> epilogues of both CTAs
  uint64_t acc_empty[kFp8Units];          // leader only: epilogue warps of both CTAs -> issuer
  uint64_t scale_full[kFp8ScaleSlots], scale_empty[kFp8ScaleSlots];
  uint32_t tmem_base;
  volatile int32_t abort_flag;
};

struct Fp8Params {
  CUtensorMap map_w[2];           // boxes of 128 and 64 rows
  CUtensorMap map_x[4];           // boxes of 128, 64, 32 and 16 rows
  const int32_t* ends;
  int32_t experts, rows;
  int32_t n;                      // channels
  int32_t col_tiles;              // of an expert's channels
  int32_t groups;                 // of k: stages
  int32_t blocks;                 // of channels (gated: of the gate's)
  uint32_t idesc;
  const float *x_scales, *w_scales;
  DenseEpilogue epi;
  int32_t* status;
  int64_t timeout_ns;
};

constexpr int kFp8Smem = 227 * 1024;
constexpr int kFp8Place = 1024;
constexpr int kFp8PlanAt = kFp8Place + kFp8Stages * kFp8Stage;
constexpr int kFp8TurnAt = kFp8PlanAt + (sizeof(GroupPlan) + 15) / 16 * 16;
static_assert(sizeof(Fp8Control) <= kFp8Place, "control block");
constexpr int kFp8ScalesAt = kFp8TurnAt + kFp8EpiWarps * kFp8Turn;
static_assert(kFp8ScalesAt + kFp8ScaleSlots * sizeof(Fp8Scales) + 1024 <= kFp8Smem, "shared memory of a CTA");

struct Fp8Tile {
  int expert, channel0;
  int first, valid;               // rows, of the pair
};
// The first `whole` tiles, then the two halves of each of the others
template <bool kGate>
__device__ __forceinline__ Fp8Tile fp8_tile_at(const Fp8Params& p, const GroupPlan& plan, int t, int whole) {
  Fp8Tile g;
  if (t >= whole) t = whole + (t - whole) / 2;
  g.expert = expert_of(plan, p.experts, t);
  const int start = plan.start[g.expert], count = plan.start[g.expert + 1] - start, parts = (count + 2 * kGroupRows - 1) / (2 * kGroupRows);
  const int in = t - plan.tile[g.expert], at = in % parts * 2 * kGroupRows;
  g.channel0 = in / parts * (kGate ? kFp8Cols / 2 : kFp8Cols);
  g.first = start + at, g.valid = min(count - at, 2 * kGroupRows);
  return g;
}
// Which accumulator's columns the warps of a side have: of a whole tile all of their own one, of half a tile 64 of the only one (gated: 32 of the gate's and
// 32 of the up rows').  Blocks of 32 columns, two or four; the channel behind the tile's first that the b-th begins with.
template <bool kGate, bool kWhole>
__device__ __forceinline__ int fp8_column(int side, int b) { return kWhole ? 32 * b : kGate ? 64 * b + 32 * side : 64 * side + 32 * b; }
template <bool kGate>
__device__ __forceinline__ int fp8_channel(int side, int b) { return 64 * side + 32 * (b & 1) + (kGate ? 0 : (b >> 1) * kFp8Unit); }
template <bool kGate>
__device__ __forceinline__ int fp8_half_channel(int side, int b, int h) { return 64 * h + (kGate ? 32 * side : kFp8Unit * side + 32 * b); }

// as mbar_arrive_pair, for two
__device__ __forceinline__ void arrive_twice(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0], 2;" ::"r"(bar) : "memory");
}

// tc_ld_wait, behind which alone v is used
__device__ __forceinline__ void wait_for(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
}

// of a CTA's 128 rows, rounded up to the smallest box
__device__ __forceinline__ int fp8_rows_staged(int valid, int cta) { return min(max(valid - cta * kGroupRows + 15, 0), kGroupRows) & ~15; }

__device__ __forceinline__ void fp8_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// a wait that ends as soon as it can: a thread that the hardware has put to sleep wakes up late, which is worth a tenth of a group's time here
__device__ __forceinline__ bool poll(DenseWaiter& w, uint32_t bar, uint32_t parity) {
  for (uint32_t spin = 0;; ++spin) {
    if (__any_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    // every 1024th probe as `late` wants it: the first sets the limit
    if ((spin & 1023u) == 1023u && __any_sync(0xffffffffu, w.late(spin == 1023u ? 63u : 64u, 1))) return false;
  }
}

// Where the phase has mostly completed: two probes, then as everybody waits, by a waiter of its own, which takes no registers meanwhile
__device__ __forceinline__ bool probe_then_wait(const Fp8Params& p, Fp8Control* ctl, uint32_t bar, uint32_t parity) {
  bool there = mbar_try_wait(bar, parity);
  if (!there) there = mbar_try_wait(bar, parity);
  if (__all_sync(0xffffffffu, there)) return true;
  DenseWaiter slow{{&ctl->abort_flag, p.status, 0, kStatusGrouped + 1, static_cast<int>(threadIdx.x >> 5)}, p.timeout_ns};
  return slow.wait_uniform(bar, parity);
}

template <bool kGate>
__global__ void __launch_bounds__(kFp8Threads, 1) fp8_pair_kernel(const __grid_constant__ Fp8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in both CTAs
  Fp8Control* ctl = reinterpret_cast<Fp8Control*>(smem);
  uint8_t* stages = smem + kFp8Place;
  GroupPlan* plan = reinterpret_cast<GroupPlan*>(smem + kFp8PlanAt);
  Fp8Scales* scales = reinterpret_cast<Fp8Scales*>(smem + kFp8ScalesAt);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int cta = static_cast<int>(cluster_ctarank());
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) prefetch_map(&p.map_w[i]);
    for (int i = 0; i < 4; ++i) prefetch_map(&p.map_x[i]);
    for (int i = 0; i < kFp8Stages; ++i) {
      mbar_init(smem_u32(&ctl->full[i]), 1);
      mbar_init(smem_u32(&ctl->empty[i]), 1);
    }
    for (int i = 0; i < kFp8Units; ++i) {
      mbar_init(smem_u32(&ctl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[i]), 2 * kFp8EpiWarps);
    }
    for (int i = 0; i < kFp8ScaleSlots; ++i) {
      mbar_init(smem_u32(&ctl->scale_full[i]), 32);
      mbar_init(smem_u32(&ctl->scale_empty[i]), kFp8EpiWarps);
    }
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kFp8EpiWarps + 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                       // the peer's barriers are initialised before anything arrives on them
  tc_fence_after();
  chain_wait();                             // nothing above touches global memory
  chain_release();                          // in this order: what precedes this launch is complete when the next one starts
  int tiles = make_plan(plan, p.ends, p.experts, p.rows, 2 * kGroupRows, p.col_tiles, p.status), whole = tiles;
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  const int step = gridDim.x / 2;
  if (2 * (tiles % step) <= step) whole = tiles / step * step, tiles += tiles - whole;      // the last turn by halves
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusGrouped + 1, warp}, p.timeout_ns};
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]);
  {
    const int64_t row_bytes = p.epi.ld_out * (p.epi.out_type == kDenseFp32 ? 4 : 2), used = plan->start[p.experts];
    clear_bytes(static_cast<char*>(p.epi.out) + used * row_bytes, (p.rows - used) * row_bytes);
  }

  if (warp < kFp8EpiWarps) {
    // --------------------------------------------------------------------------------------------- epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp8Registers));
    const int quadrant = warp & 3;                    // of the TMEM lanes: the one this warp may read
    const int side = warp >> 2;
    const uint32_t leader_empty = map_to_cta(smem_u32(&ctl->acc_empty[0]), 0);
    const uint32_t lanes = static_cast<uint32_t>(quadrant * 32) << 16;
    uint8_t* turn = smem + kFp8TurnAt + warp * kFp8Turn;
    const uint32_t full = smem_u32(&ctl->acc_full[0]), sums = tmem_base + lanes;
    uint32_t batch = 0, phase = 0, unit = side;       // the accumulator whose turn it is
    const auto wait = [&](uint32_t bar, uint32_t parity) { return probe_then_wait(p, ctl, bar, parity); };
    const auto tile = [&](auto all, int t) {           // a whole one, or half of one
      constexpr bool kWhole = all.value;
      constexpr int kBlocks = kWhole ? 4 : 2;            // of 32 columns; gated: the gate's, then the up rows'
      float sum[kBlocks][32] = {};
      uint32_t v[2][16];                                // 16 columns on their way while 16 are added
      const auto fetch = [&](int c) { tc_ld16(sums + kFp8Unit * unit + fp8_column<kGate, kWhole>(side, c >> 1) + 16 * (c & 1), v[c & 1]); };
      if (!wait(full + 8 * unit, phase)) return false;
      tc_fence_after();
      fetch(0);
      for (int left = p.groups; left > 0; ++batch) {
        if (!wait(smem_u32(&ctl->scale_full[batch % kFp8ScaleSlots]), (batch / kFp8ScaleSlots) & 1u)) return false;
        uint32_t x_at = smem_u32(&scales[batch % kFp8ScaleSlots].x[0][quadrant * 32 + lane]), w_at = smem_u32(&scales[batch % kFp8ScaleSlots].w[0][4 * side]);
        const int behind = max(left - kFp8Batch, 0);
        do {
          float x_now, w0, w1, w2, w3;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x_now) : "r"(x_at));
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w0), "=f"(w1), "=f"(w2), "=f"(w3) : "r"(w_at));
          const float scale[4] = {x_now * w0, x_now * w1, x_now * w2, x_now * w3};
          const auto add = [&](int c) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float& to = sum[c >> 1][16 * (c & 1) + i];
              to = fmaf(__uint_as_float(v[c & 1][i]), scale[c >> 1], to);
            }
          };
          wait_for(v[0]);
#pragma unroll
          for (int c = 1; c < 2 * kBlocks; ++c) {
            fetch(c);
            add(c - 1);
            wait_for(v[c & 1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (kWhole) arrive_twice(leader_empty + 8 * unit);
            else mbar_arrive_pair(leader_empty + 8 * unit);
          }
          unit = kWhole ? unit ^ 2u : (unit + 1) % kFp8Units;
          phase ^= (kWhole ? unit < 2 : unit == 0) ? 1u : 0u;          // a phase has all accumulators
          if (--left > 0) {                              // the next group's first columns
            if (!wait(full + 8 * unit, phase)) return false;
            tc_fence_after();
            fetch(0);
          }
          add(2 * kBlocks - 1);
          x_at += sizeof(scales->x[0]), w_at += sizeof(scales->w[0]);
        } while (left > behind);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->scale_empty[batch % kFp8ScaleSlots]));
      }
      // ---- results: 64 neighbouring channels of every row, or (half a gated tile) 32
      const Fp8Tile g = fp8_tile_at<kGate>(p, *plan, t, whole);
      const int row0 = g.first + cta * kGroupRows + quadrant * 32, rows = g.valid - cta * kGroupRows - quadrant * 32;      // of this warp
      if (rows <= 0) return true;
      const bool dense_rows = p.epi.out_type == kDenseFp32 ? p.n % 4 == 0 : p.n % 8 == 0;
#pragma unroll
      for (int run = 0; run < (kGate ? 1 : kBlocks / 2); ++run) {
        constexpr int kRun = kGate ? 16 * kBlocks : 64;
        const int first = g.channel0 + (kWhole ? fp8_channel<kGate>(side, 2 * run) : fp8_half_channel<kGate>(side, 0, (t - whole) & 1));
        const int count = min(kRun, p.n - first);
        if (count <= 0) continue;
        const auto put = [&](auto* out) {
          using T = std::remove_pointer_t<decltype(out)>;
          constexpr int kEach = 16 / sizeof(T), kPart = 128 / sizeof(T), kStride = 144;       // 144: no two of eight rows in one bank
          // of channel first + j; no branch in it, so that the activations run beside each other: a tile of 2048 k's 13.3 -> 11.4 us
          const auto value = [&](int j) {
            const float f = sum[2 * run + (j >> 5)][j & 31];
            if constexpr (!kGate) return f;
            const float u = sum[kBlocks / 2 + (j >> 5)][j & 31];
            if constexpr (sizeof(T) == 4) return gated_value_fp32(f, u, p.epi.clamp);
            else return gated_value(f, u, p.epi.clamp);
          };
          out += (int64_t)row0 * p.epi.ld_out + first;
#pragma unroll
          for (int part = 0; part < (kRun + kPart - 1) / kPart; ++part) {     // 128 bytes of every row
            __syncwarp();                                 // what was there has been read
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (part * kPart + j * kEach >= kRun) break;
              __align__(16) T piece[kEach];
#pragma unroll
              for (int i = 0; i < kEach; ++i) piece[i] = from_float<T>(value(part * kPart + j * kEach + i));
              *reinterpret_cast<uint4*>(turn + lane * kStride + 16 * j) = *reinterpret_cast<const uint4*>(piece);
            }
            __syncwarp();
            T* to = out + part * kPart;
            const int left = count - part * kPart;
            if (dense_rows) {
              const int at = (lane & 7) * kEach;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int r = 4 * i + (lane >> 3);
                if (r < rows && at < left) *reinterpret_cast<uint4*>(to + r * p.epi.ld_out + at) = *reinterpret_cast<const uint4*>(turn + r * kStride + 16 * (lane & 7));
              }
            } else {                                      // rows that start anywhere: a lane per column
              for (int r = 0; r < min(rows, 32); ++r)
                for (int at = lane; at < min(left, kPart); at += 32) to[r * p.epi.ld_out + at] = reinterpret_cast<const T*>(turn + r * kStride)[at];
            }
          }
        };
        if (p.epi.out_type == kDenseBf16) put(static_cast<__nv_bfloat16*>(p.epi.out));
        else if (p.epi.out_type == kDenseFp16) put(static_cast<__half*>(p.epi.out));
        else put(static_cast<float*>(p.epi.out));
      }
      return true;
    };
    bool ok = true;
    int t = blockIdx.x / 2;
    for (; ok && t < whole; t += step) ok = tile(std::true_type(), t);
    if (ok && t < tiles) {
      unit &= 2u;                                      // both sides go on with the first of the two whose turn it is
      tile(std::false_type(), t);
    }
    tc_ld_wait();                                       // one that was abandoned may have columns on their way
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8FewRegisters));
    if (warp == kFp8EpiWarps) {
      // --------------------------------------------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t leader_full0 = map_to_cta(full0, 0), base = smem_u32(stages);
      bool ok = true;
      for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
        const Fp8Tile g = fp8_tile_at<kGate>(p, *plan, t, whole);
        const int rows = fp8_rows_staged(g.valid, cta), x_row = g.first + cta * kGroupRows;
        const bool all = t < whole;
        const uint32_t tx = (fp8_rows_staged(g.valid, 0) + fp8_rows_staged(g.valid, 1)) * 128 + 2 * (all ? 2 * kFp8StageHalf : kFp8StageHalf);
        const int w_row = g.channel0 + (kGate ? 0 : cta * kFp8Unit) + (all ? 0 : ((t - whole) & 1) * (kFp8Unit / 2)), part = kGate ? cta : 0;
        for (int kb = 0; kb < p.groups; ++kb) {
          if (!waiter.wait_uniform(empty0 + 8 * stage, phase ^ 1u)) { ok = false; break; }
          const uint32_t bar = leader_full0 + 8 * stage, a = base + stage * kFp8Stage;
          if (elect_one()) {
            if (cta == 0) mbar_expect_tx(full0 + 8 * stage, tx);
            pair_load_4d(a + kFp8StageA, &p.map_w[all ? 0 : 1], kb * 128, w_row, part, g.expert, bar);
            int done = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (rows & (128 >> i)) {
                pair_load_2d(a + done * 128, &p.map_x[i], kb * 128, x_row + done, bar);
                done += 128 >> i;
              }
          }
          __syncwarp();
          if (++stage == kFp8Stages) { stage = 0; phase ^= 1u; }
        }
      }
    } else if (warp == kFp8EpiWarps + 1) {
      // --------------------------------------------------------------------------------------------- issuer
      if (cta == 0) {
        int stage = 0;
        uint32_t phase = 0, it = 0;
        const uint32_t lo0 = (smem_u32(stages) & 0x3FFFFu) >> 4;
        const uint64_t hi = operand_desc(false, 0);
        const auto issue = [&](auto halves) {              // one tile, or half of one
          for (int kb = 0; kb < p.groups; ++kb) {
            if (!poll(waiter, full0 + 8 * stage, phase)) return false;
#pragma unroll
            for (int h = 0; h < halves.value; ++h, ++it) {
              const uint32_t acc = it % kFp8Units;
              if (!poll(waiter, smem_u32(&ctl->acc_empty[acc]), ((it / kFp8Units) & 1u) ^ 1u)) return false;
              tc_fence_after();
              const uint32_t a = lo0 + stage * (kFp8Stage >> 4), b = a + ((kFp8StageA + h * kFp8StageHalf) >> 4), d = tmem_base + acc * kFp8Unit;
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) fp8_product(d, hi | (a + 2 * k), hi | (b + 2 * k), p.idesc, k != 0 ? 1u : 0u);
                if (h == halves.value - 1) pair_commit(empty0 + 8 * stage);
                pair_commit(smem_u32(&ctl->acc_full[acc]));
              }
            }
            __syncwarp();
            if (++stage == kFp8Stages) { stage = 0; phase ^= 1u; }
          }
          return true;
        };
        bool ok = true;
        int t = blockIdx.x / 2;
        for (; ok && t < whole; t += step) ok = issue(std::integral_constant<int, 2>());
        if (ok && t < tiles) issue(std::integral_constant<int, 1>());
      }
    } else if (warp == kFp8EpiWarps + 2) {
      // ------------------------------------------------------------------------------------------- scales
      uint32_t batch = 0;
      bool ok = true;
      const int group = lane & 7, row0 = lane >> 3;      // a lane's group of a batch, and the first of its rows: eight lanes read 32 bytes of a row
      for (int t = blockIdx.x / 2; ok && t < tiles; t += step) {
        const Fp8Tile g = fp8_tile_at<kGate>(p, *plan, t, whole);
        const int rows = g.valid - cta * kGroupRows;
        const float* x = p.x_scales + (int64_t)(g.first + cta * kGroupRows + row0) * p.groups + group;
        // blocks row0 and row0 + 4 of the eight: those of either side
        const float* w[2];
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const int up = !kGate ? 0 : t < whole ? row0 >> 1 : row0 & 1;
          const int channel = g.channel0 + (t < whole ? fp8_channel<kGate>(side, row0) : fp8_half_channel<kGate>(side, row0 & 1, (t - whole) & 1));
          w[side] = p.w_scales + (((int64_t)g.expert * (kGate ? 2 : 1) + up) * p.blocks + min(channel / kScaleBlock, p.blocks - 1)) * p.groups + group;
        }
        for (int kb = 0; kb < p.groups; kb += kFp8Batch, ++batch) {
          if (!waiter.wait_uniform(smem_u32(&ctl->scale_empty[batch % kFp8ScaleSlots]), ((batch / kFp8ScaleSlots) & 1u) ^ 1u)) { ok = false; break; }
          Fp8Scales& to = scales[batch % kFp8ScaleSlots];
          const bool there = kb + group < p.groups;
#pragma unroll
          for (int i = 0; i < 2; ++i) copy_word(smem_u32(&to.w[group][4 * i + row0]), there ? w[i] + kb : p.w_scales, there);
          const int last = there ? rows - row0 : 0;
#pragma unroll 8
          for (int r = 0; r < kGroupRows; r += 4) copy_word(smem_u32(&to.x[group][r + row0]), r < last ? x + (int64_t)r * p.groups + kb : p.x_scales, r < last);
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl->scale_full[batch % kFp8ScaleSlots])) : "memory");
        }
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
  if (warp == kFp8EpiWarps + 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
}

// ---------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------
template <typename F>
cudaError_t for_each_fp8_kernel(F f) {
  const cudaError_t e = f(fp8_pair_kernel<false>, false);
  return e == cudaSuccess ? f(fp8_pair_kernel<true>, true) : e;
}

cudaError_t launch_fp8_pairs(const GroupedProduct& p, int sms, cudaStream_t s) {
  Fp8Params d = {};
  const bool gate = p.kind == kGated;
  d.ends = p.ends, d.experts = p.experts, d.rows = p.rows, d.n = p.n;
  const int width = gate ? kFp8Cols / 2 : kFp8Cols;
  d.col_tiles = (p.n + width - 1) / width;
  d.groups = (p.k + kScaleBlock - 1) / kScaleBlock;
  d.blocks = (p.n + kScaleBlock - 1) / kScaleBlock;
  d.idesc = product_idesc(kDenseFp16, false, false, 2 * kGroupRows, kFp8Unit);         // format 0: FP16, or in 8 bits E4M3
  d.x_scales = p.x_scales, d.w_scales = p.w_scales;
  d.epi = p.epi;
  d.status = p.status;
  d.timeout_ns = (p.timeout_ms > 0 ? (int64_t)p.timeout_ms : 2000) * 1000000ll;
  const uint64_t n = p.n, k = p.k, parts = gate ? 2 : 1;
  bool ok = true;
  for (int i = 0; ok && i < 2; ++i)
    ok = encode_map(&d.map_w[i], kGroupedE4m3, p.w, 4, {k, n, parts, static_cast<uint64_t>(p.experts), 1}, {k, n * k, parts * n * k, 0}, {128, 128u >> i, 1, 1, 1});
  for (int i = 0; ok && i < 4; ++i)
    ok = encode_map(&d.map_x[i], kGroupedE4m3, p.x, 2, {k, static_cast<uint64_t>(p.rows), 1, 1, 1}, {static_cast<uint64_t>(p.x_ld), 0, 0, 0}, {128, 128u >> i, 1, 1, 1});
  const int64_t most = ((int64_t)p.rows / (2 * kGroupRows) + std::min(p.experts, p.rows)) * d.col_tiles;
  if (!ok || most > INT32_MAX / 2) return cudaErrorInvalidValue;
  const int grid = 2 * static_cast<int>(std::min<int64_t>(sms / 2, 2 * most));       // every tile could come in halves
  return for_each_fp8_kernel([&](auto kernel, bool k_gate) { return k_gate != gate ? cudaSuccess : launch_clustered(kernel, dim3(grid), dim3(kFp8Threads), kFp8Smem, 2, s, d); });
}

// ---------------------------------------------------------------------------------------------------------------------
// Quantiser: s = max|x| / 448 for each 128 values of a row, q = x / s rounded to the nearest E4M3 value, ties to even.
// Eight lanes have a group, sixteen values each, which stay in registers between the maximum and the quotients.
// What bounds it is instructions, 4 of 5 issue slots: 3840 x 2304 in FP16 (27 MB) 8.2 us, 3840 x 5120 in BF16 16.6, 23040 x 5120 83.7 (4.3 TB/s); 7 rows 2.6, the
// launch.  With a look at every quotient's dropped bits instead of rounding it twice, and all sixteen divided where one is on a border: 12.5, 27.6 and 151 us;
// in BF16 quotients on a border are common, as s is a number of eight bits by 7.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 256, kQuantLanes = 8, kQuantEach = kScaleBlock / kQuantLanes;

// x / s within a step, with its last bit set where it is not exact, so that it rounds to fewer bits as the exact quotient does: remainders are exact in
// one fma.  inv is the rounded reciprocal, or (kDivide) of no use.
template <bool kDivide>
__device__ __forceinline__ float odd_quotient(float x, float s, float inv) {
  float q;
  if (kDivide) {
    q = __fdiv_rn(x, s);
  } else {
    q = x * inv;
    q = fmaf(fmaf(-q, s, x), inv, q);
  }
  const float rest = fmaf(-q, s, x);
  uint32_t bits = __float_as_uint(q);
  if (rest != 0.f) {
    if ((rest < 0.f) != (x < 0.f)) --bits;       // towards zero (a q that is one, where the quotient leaves the numbers, has all of x left and stays) ...
    bits |= 1u;                                  // ... and marked
  }
  return __uint_as_float(bits);
}
__device__ __forceinline__ uint32_t two_e4m3(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ __half2 larger_of(__half2 top, __half2 v) { return __hmax2_nan(top, __habs2(v)); }
__device__ __forceinline__ __nv_bfloat162 larger_of(__nv_bfloat162 top, __nv_bfloat162 v) { return __hmax2_nan(top, __habs2(v)); }
__device__ __forceinline__ float2 two_values(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 two_values(__nv_bfloat162 v) { return __bfloat1622float2(v); }
template <typename T> struct TwoOf;
template <> struct TwoOf<__half> { using type = __half2; };
template <> struct TwoOf<__nv_bfloat16> { using type = __nv_bfloat162; };

// kVec: eight neighbouring values in one load; else (widths, strides or places that do not allow it) one.  kFlat: rows follow each other in whole groups,
// so that the place of a group is its number.
template <typename T, bool kVec, bool kFlat>
__global__ void __launch_bounds__(kQuantThreads) quantize_fp8_kernel(const T* x, int64_t ld, uint8_t* q, float* scales, uint32_t total, uint32_t groups, int k) {
  chain_wait();
  chain_release();
  using P = typename TwoOf<T>::type;
  const uint64_t index = (uint64_t)blockIdx.x * (kQuantThreads / kQuantLanes) + threadIdx.x / kQuantLanes;
  const bool there = index < total;            // eight lanes alike
  const int lane = threadIdx.x % kQuantLanes;
  int64_t row = 0;
  int first = 0, count = there ? kScaleBlock : 0;
  if (!kFlat) {
    const uint32_t r = static_cast<uint32_t>(index) / groups;
    row = r, first = static_cast<int>(static_cast<uint32_t>(index) - r * groups) * kScaleBlock;
    count = there ? min(kScaleBlock, k - first) : 0;
  }
  const T* in = x + (kFlat ? (int64_t)index * kScaleBlock : row * ld + first);
  uint8_t* out = q + (kFlat ? (int64_t)index * kScaleBlock : row * k + first);
  // value j of a lane: kVec: eight neighbours from 8 lane on, and eight from 64 + 8 lane on; else every eighth from lane on
  P v[kQuantEach / 2];
  if constexpr (kVec) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 f = make_uint4(0u, 0u, 0u, 0u);
      if (64 * h + 8 * lane < count) f = *reinterpret_cast<const uint4*>(in + 64 * h + 8 * lane);
      *reinterpret_cast<uint4*>(v + 4 * h) = f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kQuantEach / 2; ++j) {
      const int a = lane + 16 * j, b = a + 8;
      v[j] = P{a < count ? in[a] : T(0.f), b < count ? in[b] : T(0.f)};
    }
  }
  P top2 = {T(0.f), T(0.f)};
#pragma unroll
  for (int j = 0; j < kQuantEach / 2; ++j) top2 = larger_of(top2, v[j]);
  // magnitudes as bits: NaN is above infinity there, so neither is lost
  const float2 both = two_values(top2);
  uint32_t top = max(__float_as_uint(both.x), __float_as_uint(both.y)) & 0x7fffffffu;
#pragma unroll
  for (int d = kQuantLanes / 2; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  const bool finite = top < 0x7f800000u;
  const float s = !finite ? __uint_as_float(0x7fffffffu) : top == 0 ? 1.f : __fdiv_rn(__uint_as_float(top), 448.f);
  if (there && lane == 0) scales[index] = s;
  // remainders of quotients by a very small scale would be no numbers, and neither would its reciprocal
  const bool tiny = s < 0x1p-60f;
  // The products with the reciprocal are within 2^-22 of the quotients: where a little more and a little less round alike, so does the quotient.  Where
  // they do not, mostly on a border itself (whose last bit decides), the two values are divided.
  const float inv = __fdiv_rn(1.f, s), more = inv * (1.f + 0x1p-21f), less = inv * (1.f - 0x1p-21f);
  uint32_t b[kQuantEach / 2];
#pragma unroll
  for (int j = 0; j < kQuantEach / 2; ++j) {
    const float2 f = two_values(v[j]);
    b[j] = two_e4m3(f.x * more, f.y * more);
    if (b[j] != two_e4m3(f.x * less, f.y * less)) b[j] = two_e4m3(odd_quotient<false>(f.x, s, inv), odd_quotient<false>(f.y, s, inv));
  }
  if (tiny) {
#pragma unroll
    for (int j = 0; j < kQuantEach / 2; ++j) {
      const float2 f = two_values(v[j]);
      b[j] = two_e4m3(odd_quotient<true>(f.x * 0x1p80f, s * 0x1p80f, 0.f), odd_quotient<true>(f.y * 0x1p80f, s * 0x1p80f, 0.f));
    }
  }
  if (!finite) {
#pragma unroll
    for (uint32_t& w : b) w = 0;
  }
  if constexpr (kVec) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (64 * h + 8 * lane < count) *reinterpret_cast<uint2*>(out + 64 * h + 8 * lane) = make_uint2(b[4 * h] | b[4 * h + 1] << 16, b[4 * h + 2] | b[4 * h + 3] << 16);
  } else {
#pragma unroll
    for (int j = 0; j < kQuantEach / 2; ++j) {
      const int a = lane + 16 * j;
      if (a < count) out[a] = static_cast<uint8_t>(b[j] & 0xffu);
      if (a + 8 < count) out[a + 8] = static_cast<uint8_t>(b[j] >> 8);
    }
  }
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t ld, uint8_t* q, float* scales, int m, int k, cudaStream_t s) {
  const T* in = static_cast<const T*>(x);
  const bool vec = k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const bool flat = vec && k % kScaleBlock == 0 && (ld == k || m == 1);
  const uint32_t groups = (static_cast<uint32_t>(k) + kScaleBlock - 1) / kScaleBlock;
  const uint64_t total = (uint64_t)m * groups, blocks = (total + kQuantThreads / kQuantLanes - 1) / (kQuantThreads / kQuantLanes);
  if (total > UINT32_MAX || blocks > INT32_MAX) return cudaErrorInvalidValue;
  const uint32_t n = static_cast<uint32_t>(total);
  const auto kernel = flat ? quantize_fp8_kernel<T, true, true> : vec ? quantize_fp8_kernel<T, true, false> : quantize_fp8_kernel<T, false, false>;
  return launch_chained(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kQuantThreads), 0, s, in, ld, q, scales, n, groups, k);
}

}  // namespace

cudaError_t prepare_fp8() {
  return for_each_fp8_kernel([](auto kernel, bool) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8Smem); });
}

cudaError_t launch_fp8(const GroupedProduct& p, cudaStream_t s) {
  const int sms = dense_sms();
  if (sms == 0) return cudaErrorNotReady;
  const ChainScope chain(true);
  return grouped_few_rows(p, sms) ? launch_grouped_few(p, sms, s) : launch_fp8_pairs(p, sms, s);
}

cudaError_t launch_quantize_fp8(const void* x, int type, int64_t ld, uint8_t* q, float* scales, int m, int k, cudaStream_t s) {
  if (m <= 0) return cudaSuccess;
  const ChainScope chain(true);
  return type == kDenseBf16 ? launch_quantize<__nv_bfloat16>(x, ld, q, scales, m, k, s) : launch_quantize<__half>(x, ld, q, scales, m, k, s);
}

}  // namespace mmoe
