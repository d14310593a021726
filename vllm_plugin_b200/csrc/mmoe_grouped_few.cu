// Products of a layer's experts with few rows each, for sm_100a (see mmoe_grouped.cuh).
#include <algorithm>

#include "mmoe_grouped_device.cuh"

namespace mmoe {

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// Bound by the bytes of the weights: a CTA has 128 rows of an expert's weights (operand A; gated: 64 gate and 64 up rows) and up to 64 of its rows
// (operand B, padded to 16), so that a handful of rows costs what their weights cost.  Two CTAs to an SM.  Where that leaves SMs without one, K
// is split over the CTAs of a cluster, whose partial sums meet in shared memory in the order of the CTAs, as those of the dense products
// of few tokens do: no atomics, no workspace, the same bits in every call.  h is rounded to its type, as on pairs.  The grid has a CTA for every tile there could be; which one it is follows
// from `ends`, and those beyond the last leave at once.
//
// 8 bits: a group of 128 k's goes into one of four accumulators.  Four warps, a lane for each row of weights, multiply it by its scales and add it
// to registers; the scales come word by word, up to three batches of eight groups ahead.
//
// What bounds it: bytes of the weights where there are enough of them, else a launch's start and the last bytes' latency.  6 rows of 6 experts in BF16, 5120 ->
// 2 x 2304 and 2304 -> 5120 (425 MB): 74 us for both in turn, 5.7 TB/s.  8 bits: 384 rows of 41 experts, 5120 -> 2 x 2304 (0.97 GB) 158 us, 6.1 TB/s; one row,
// 2304 -> 5120 (12 MB) 6.1 us, where its bytes are 1.8.  Tried: eight warps that read the sums, and one CTA to an SM with
// twice the stages: no gain.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = kGroupRows;                  // rows of A
constexpr int kFewCols = 64;                          // most rows of B
constexpr int kFewStageA = kFewRows * 128, kFewStage = kFewStageA + kFewCols * 128;
constexpr int kFewStages = 4;
constexpr int kFewThreads = 256;                      // producer, issuer, four warps that read the sums, one that fetches scales; all finish
constexpr int kFewMaxSplit = 6;
constexpr int kFewSmem = 113 * 1024;
constexpr int kFewBatch = 8, kFewSlots = 4, kFewAccumulators = 4;

struct alignas(16) FewScales {
  float x[kFewBatch][kFewCols];
  float w[kFewBatch][2];                              // gate (or only) and up rows
};
struct FewControl {
  uint64_t full[kFewStages], empty[kFewStages];
  uint64_t acc_full[kFewAccumulators], acc_empty[kFewAccumulators];
  uint64_t scale_full[kFewSlots], scale_empty[kFewSlots];
  uint64_t sums_in;                                   // what the other CTAs of the cluster send
  uint32_t tmem_base;
  volatile int32_t abort_flag;
  int32_t tile[4];                                    // expert (-1: none), block of its weights' rows, first row, rows
  int32_t used;                                       // rows of all experts
  FewScales scales[kFewSlots];
};
constexpr int kFewPlace = 10 * 1024;
static_assert(sizeof(FewControl) <= kFewPlace, "control block");
static_assert(kFewPlace + kFewStages * kFewStage + 1024 <= kFewSmem, "shared memory of a CTA");
// sums of all rows of a tile, and what the other CTAs send of those that this one finishes: of `split` CTAs each at most 1 / split, rounded up
static_assert((kFewCols + kFewCols + kFewMaxSplit) * kFewRows * 4 <= kFewStages * kFewStage, "partial sums fit where the stages were");

struct FewParams {
  CUtensorMap map_w;
  CUtensorMap map_x[3];           // boxes of 64, 32 and 16 rows
  const int32_t* ends;
  int32_t experts, rows;
  int32_t n;                      // channels
  int32_t row_tiles;              // of an expert's weights
  int32_t k_stages, split;
  int32_t blocks;                 // of channels, of 128 (gated: of the gate's)
  uint32_t idesc;                 // without the columns
  int32_t tmem_cols;
  const float *x_scales, *w_scales;
  DenseEpilogue epi;
  int32_t zero_behind;
  int32_t* status;
  int64_t timeout_ns;
};

__device__ __forceinline__ void load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

template <bool kFp8>
__device__ __forceinline__ void few_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kFp8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    single_product<false>(d, a, b, idesc, accumulate);
}

// Which tile the t-th is: by one warp.  An expert has row_tiles of them for every 64 rows that it has begun.
__device__ __forceinline__ void find_tile(const FewParams& p, int t, FewControl* ctl) {
  const int lane = threadIdx.x & 31;
  int before = 0, last = 0;                // tiles and rows of the experts in front
  bool bad = false;
  int expert = -1, in = 0, first = 0, count = 0;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    const int end = e >= p.experts ? 0 : p.ends != nullptr ? p.ends[e] : p.rows;
    int start = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) start = last;
    const bool here = e < p.experts;
    bad |= here && (end < start || end > p.rows);
    const int own = here && !bad ? (end - start + kFewCols - 1) / kFewCols * p.row_tiles : 0;
    int tiles = own;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, tiles, d);
      if (lane >= d) tiles += v;
    }
    const int from = before + tiles - own;
    const uint32_t mine = __ballot_sync(0xffffffffu, t >= from && t < from + own);
    if (mine != 0) {
      const int whose = __ffs(mine) - 1;
      expert = e0 + whose, in = t - __shfl_sync(0xffffffffu, from, whose);
      first = __shfl_sync(0xffffffffu, start, whose), count = __shfl_sync(0xffffffffu, end, whose) - first;
    }
    before += __shfl_sync(0xffffffffu, tiles, 31);
    last = __shfl_sync(0xffffffffu, end, min(31, p.experts - 1 - e0));
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    if (bad && blockIdx.x == 0) report_bad_index(p.status);
    const int parts = max(1, (count + kFewCols - 1) / kFewCols), width = ((count + parts - 1) / parts + 15) & ~15, at = in % parts * width;
    ctl->tile[0] = bad ? -1 : expert, ctl->tile[1] = in / parts, ctl->tile[2] = first + at, ctl->tile[3] = min(count - at, width);
    ctl->used = bad ? 0 : last;
  }
}

template <bool kFp8, bool kGate>
__global__ void __launch_bounds__(kFewThreads, 2) grouped_few_kernel(const __grid_constant__ FewParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the same offset in all CTAs
  FewControl* ctl = reinterpret_cast<FewControl*>(smem);
  uint8_t* stages = smem + kFewPlace;
  constexpr int kDepth = kFp8 ? 128 : 64;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int k0 = static_cast<int>((int64_t)p.k_stages * rank / p.split), k1 = static_cast<int>((int64_t)p.k_stages * (rank + 1) / p.split);
  if (threadIdx.x == 0) {
    prefetch_map(&p.map_w);
    for (int i = 0; i < 3; ++i) prefetch_map(&p.map_x[i]);
    for (int i = 0; i < kFewStages; ++i) {
      mbar_init(smem_u32(&ctl->full[i]), 1);
      mbar_init(smem_u32(&ctl->empty[i]), 1);
    }
    for (int i = 0; i < kFewAccumulators; ++i) {
      mbar_init(smem_u32(&ctl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[i]), 4);
    }
    for (int i = 0; i < kFewSlots; ++i) {
      mbar_init(smem_u32(&ctl->scale_full[i]), 32);
      mbar_init(smem_u32(&ctl->scale_empty[i]), 4);
    }
    mbar_init(smem_u32(&ctl->sums_in), 1);
    ctl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  chain_wait();                             // nothing above touches global memory
  chain_release();                          // in this order: what precedes this launch is complete when the next one starts
  if (warp == 0) find_tile(p, blockIdx.x / p.split, ctl);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t full0 = smem_u32(&ctl->full[0]), empty0 = smem_u32(&ctl->empty[0]), base = smem_u32(stages);
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  const int expert = ctl->tile[0], block = ctl->tile[1], first = ctl->tile[2], valid = ctl->tile[3];
  DenseWaiter waiter{{&ctl->abort_flag, p.status, 0, kStatusGrouped + 2, warp}, p.timeout_ns};
  if (p.zero_behind) {
    const int64_t row_bytes = p.epi.ld_out * (p.epi.out_type == kDenseFp32 ? 4 : 2);
    clear_bytes(static_cast<char*>(p.epi.out) + ctl->used * row_bytes, (p.rows - ctl->used) * row_bytes);
  }

  if (expert >= 0) {                        // the same in all CTAs of the cluster
    const int cols = (valid + 15) & ~15;
    const uint32_t acc_stride = kFp8 ? kFewCols : 0;
    if (warp == 0) {
      // ------------------------------------------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 0;
      const int w_row = block * (kGate ? kFewRows / 2 : kFewRows);
      for (int kb = k0; kb < k1; ++kb) {
        if (!waiter.wait_uniform(empty0 + 8 * stage, phase ^ 1u)) break;
        const uint32_t bar = full0 + 8 * stage, w = base + stage * kFewStage;
        if (elect_one()) {
          mbar_expect_tx(bar, kFewStageA + cols * 128);
          load_4d(w, &p.map_w, kb * kDepth, w_row, 0, expert, bar);
          if (kGate) load_4d(w + 8192, &p.map_w, kb * kDepth, w_row, 1, expert, bar);
          int done = 0;
#pragma unroll
          for (int i = 0; i < 3; ++i)
            if (cols & (64 >> i)) {
              tma_load_2d(w + kFewStageA + done * 128, &p.map_x[i], kb * kDepth, first + done, bar);
              done += 64 >> i;
            }
        }
        __syncwarp();
        if (++stage == kFewStages) { stage = 0; phase ^= 1u; }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------------------------------- issuer
      int stage = 0;
      uint32_t phase = 0, it = 0;
      bool ok = true;
      const uint64_t hi = operand_desc(false, 0);
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(cols >> 3) << 17);
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const uint32_t acc = kFp8 ? it % kFewAccumulators : 0;
        if (kFp8 && !waiter.wait_uniform(smem_u32(&ctl->acc_empty[acc]), ((it / kFewAccumulators) & 1u) ^ 1u)) { ok = false; break; }
        if (!waiter.wait_uniform(full0 + 8 * stage, phase)) { ok = false; break; }
        tc_fence_after();
        const uint32_t w = ((base + stage * kFewStage) & 0x3FFFFu) >> 4, x = w + (kFewStageA >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            few_product<kFp8>(tmem_base + acc * acc_stride, hi | (w + 2 * k), hi | (x + 2 * k), idesc, (!kFp8 && kb > k0) || k > 0 ? 1u : 0u);
          tc_commit(empty0 + 8 * stage);
          if (kFp8) tc_commit(smem_u32(&ctl->acc_full[acc]));
        }
        __syncwarp();
        if (++stage == kFewStages) { stage = 0; phase ^= 1u; }
      }
      if (!kFp8 && ok && elect_one()) tc_commit(smem_u32(&ctl->acc_full[0]));
      __syncwarp();
    } else if (kFp8 && warp == 6) {
      // ------------------------------------------------------------------------------------------- scales
      // eight lanes copy 32 bytes of a row's scales
      const int group = lane & 7, row0 = lane >> 3;
      const float* x = p.x_scales + (int64_t)(first + row0) * p.k_stages + group;
      const int of = min(block * (kGate ? kFewRows / 2 : kFewRows) / kScaleBlock, p.blocks - 1);
      const float* w = p.w_scales + (((int64_t)expert * (kGate ? 2 : 1) + (kGate ? row0 & 1 : 0)) * p.blocks + of) * p.k_stages + group;
      uint32_t batch = 0;
      for (int kb = k0; kb < k1; kb += kFewBatch, ++batch) {
        const uint32_t slot = batch % kFewSlots;
        if (!waiter.wait_uniform(smem_u32(&ctl->scale_empty[slot]), ((batch / kFewSlots) & 1u) ^ 1u)) break;
        FewScales& to = ctl->scales[slot];
        const bool there = kb + group < k1;
        if (row0 < 2) copy_word(smem_u32(&to.w[group][row0]), there ? w + kb : p.w_scales, there);
        for (int r = row0; r < cols; r += 4) copy_word(smem_u32(&to.x[group][r]), there && r < valid ? x + (int64_t)(r - row0) * p.k_stages + kb : p.x_scales, there && r < valid);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl->scale_full[slot])) : "memory");
      }
    }

    // ----------------------------------------------------------------------------------------------- sums
    // The partial sums take the place of the stages, which this CTA needs no more when its accumulator is complete: [row][128 channels].  Each CTA
    // of the cluster finishes some of the rows; the others send it theirs, in one copy each, when no CTA needs its stages any more.
    constexpr int kRowBytes = kFewRows * 4;
    const int own = (valid + p.split - 1) / p.split, from = rank * own, mine = max(0, min(own, valid - from));
    const uint32_t came = smem_u32(&ctl->sums_in);
    uint8_t* sent = stages + cols * kRowBytes;           // [CTA, this one left out][row][128 channels]
    if (p.split > 1 && threadIdx.x == 0) mbar_expect_tx(came, (p.split - 1) * mine * kRowBytes);
    if (warp >= 2 && warp < 6) {
      const int row = (warp & 3) * 32 + lane;
      const uint32_t d = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      float* sums = reinterpret_cast<float*>(stages) + row;
      if constexpr (kFp8) {
        float sum[kFewCols] = {};
        uint32_t it = 0;
        bool ok = true;
        const int up = kGate ? row >> 6 : 0;
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const uint32_t in = it % kFewBatch, slot = it / kFewBatch % kFewSlots, acc = it % kFewAccumulators;
          if (in == 0 && !waiter.wait_warp(smem_u32(&ctl->scale_full[slot]), (it / kFewBatch / kFewSlots) & 1u, 0)) { ok = false; break; }
          if (!waiter.wait_warp(smem_u32(&ctl->acc_full[acc]), (it / kFewAccumulators) & 1u, 0)) { ok = false; break; }
          tc_fence_after();
          const FewScales& now = ctl->scales[slot];
          const float ws = now.w[in][up];
#pragma unroll
          for (int c = 0; c < kFewCols; c += 16) {
            if (c >= cols) break;
            uint32_t v[16];
            tc_ld16(d + acc * acc_stride + c, v);
            tc_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float4 xs = *reinterpret_cast<const float4*>(&now.x[in][c + j]);
              sum[c + j] = fmaf(__uint_as_float(v[j]), xs.x * ws, sum[c + j]);
              sum[c + j + 1] = fmaf(__uint_as_float(v[j + 1]), xs.y * ws, sum[c + j + 1]);
              sum[c + j + 2] = fmaf(__uint_as_float(v[j + 2]), xs.z * ws, sum[c + j + 2]);
              sum[c + j + 3] = fmaf(__uint_as_float(v[j + 3]), xs.w * ws, sum[c + j + 3]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&ctl->acc_empty[acc]));
            if (in == kFewBatch - 1 || kb == k1 - 1) mbar_arrive(smem_u32(&ctl->scale_empty[slot]));
          }
        }
        // the last group's accumulator is complete: so are all products, and nothing reads the stages any more
        if (ok) {
#pragma unroll
          for (int j = 0; j < kFewCols; ++j)
            if (j < cols) sums[j * kFewRows] = sum[j];
        }
      } else if (waiter.wait_warp(smem_u32(&ctl->acc_full[0]), 0, k1 - k0)) {
        tc_fence_after();
        for (int c = 0; c < cols; c += 16) {
          uint32_t v[16];
          tc_ld16(d + c, v);
          tc_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) sums[(c + j) * kFewRows] = __uint_as_float(v[j]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    cluster_sync_all();
    if (p.split > 1) {
      if (threadIdx.x == 0)
        for (int r = 0; r < p.split; ++r) {
          const int theirs = min(own, valid - r * own);
          if (r != rank && theirs > 0)
            cluster_send(map_to_cta(base + (cols + (rank < r ? rank : rank - 1) * own) * kRowBytes, r), base + r * own * kRowBytes, theirs * kRowBytes, map_to_cta(came, r));
        }
      __syncwarp();
      waiter.wait_warp(came, 0, 0);
      __syncwarp();
      cluster_arrive();                     // what this CTA waited for has come; behind the matching wait, all that it has sent has
    }
    constexpr int kGroups = kGate ? kFewRows / 16 : kFewRows / 8;               // eight channels each
    static_assert(kFewThreads % kGroups == 0, "a thread keeps its channels");
    const int g = static_cast<int>(threadIdx.x) % kGroups, channel = block * 8 * kGroups + 8 * g, there = p.n - channel;
    for (int i = threadIdx.x; i < mine * kGroups; i += kFewThreads) {
      const int t = i / kGroups, at = (t * kFewRows + 8 * g) * 4;
      float a[8] = {}, b[8] = {};
      for (int r = 0; r < p.split; ++r) {                // in the order of the CTAs
        const float* part = reinterpret_cast<const float*>((r == rank ? stages + from * kRowBytes : sent + (r < rank ? r : r - 1) * own * kRowBytes) + at);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a[j] += part[j];
          if (kGate) b[j] += part[kFewRows / 2 + j];
        }
      }
      if (there <= 0) continue;
      const int64_t row = first + from + t;
      if (kGate) {
        if (!kFp8 && p.epi.preact != nullptr) {
          float* keep = p.epi.preact + row * 2 * p.epi.inter + channel;
          store8(keep, a, there);
          store8(keep + p.epi.inter, b, there);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = kFp8 && p.epi.out_type == kDenseFp32 ? gated_value_fp32(a[j], b[j], p.epi.clamp) : gated_value(a[j], b[j], p.epi.clamp);
      }
      const int64_t to = row * p.epi.ld_out + channel;
      if (p.epi.out_type == kDenseBf16) store8(static_cast<__nv_bfloat16*>(p.epi.out) + to, a, there);
      else if (p.epi.out_type == kDenseFp16) store8(static_cast<__half*>(p.epi.out) + to, a, there);
      else store8(static_cast<float*>(p.epi.out) + to, a, there);
    }
    if (p.split > 1) {
      __syncwarp();
      cluster_wait();
    }
  }

  // ---------------------------------------------------------------------------------------------------- teardown
  __syncwarp();
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
// the most tiles that there can be
int64_t few_tiles(const GroupedProduct& p) {
  const int width = p.kind == kGated ? kFewRows / 2 : kFewRows;
  return (std::min(p.experts, p.rows) + (int64_t)(p.rows - 1) / kFewCols) * ((p.n + width - 1) / width);
}

// CTAs that share a tile's K, by what their stages cost (twice that where two share an SM) and what meeting costs, in clocks.  With 1, 2, 3, 4, 6 of them,
// 8 bits, 5120 -> 5120 (40 tiles): one row 15.0, 10.0, 8.4, 8.4, 8.0 us, 64 rows 24.0, 14.9, 12.7, 13.9, 13.3; 128 rows (80 tiles) 24.2, 18.8, 16.0, 23.1, -; gated
// 5120 -> 2 x 2304 (72), 128 rows, 24.4, 15.4, 16.0, 22.9, -; 2304 -> 1024 (8), one row 8.4, 6.6, 5.7, 5.3, 5.1, 64 rows 13.3, 9.6, 8.4, 7.8, 7.2.  Clusters of 7 and 8 take longer.
// The columns are those of a call of one expert; with more of them an expert's are fewer, and the cost of a stage is taken to be too high.
int few_split(const GroupedProduct& p, int64_t tiles, int k_stages, int sms) {
  const int cols = std::min((p.rows + 15) & ~15, kFewCols);
  const int64_t stage = p.type == kGroupedE4m3 ? 475 + 6 * cols : 340 + cols;
  int64_t least = INT64_MAX;
  int best = 1;
  for (int c : {1, 2, 3, 4, kFewMaxSplit}) {
    if (c > 1 && (tiles * c > 2 * sms || c > k_stages)) break;
    const int64_t cost = (k_stages + c - 1) / c * stage * (tiles * c <= sms ? 1 : 2) + 8 * cols * c;
    if (cost < least) least = cost, best = c;
  }
  return best;
}

template <typename F>
cudaError_t for_each_few_kernel(F f) {
  cudaError_t e = f(grouped_few_kernel<false, false>, false, false);
  if (e == cudaSuccess) e = f(grouped_few_kernel<false, true>, false, true);
  if (e == cudaSuccess) e = f(grouped_few_kernel<true, false>, true, false);
  if (e == cudaSuccess) e = f(grouped_few_kernel<true, true>, true, true);
  return e;
}

}  // namespace

// Against pairs.  16 bits, 5120 x 5120 of one expert: 16 rows 17.6 -> 10.4 us, 64 18.4 -> 12.1, 128 19.3 -> 16.0, 192 (120 tiles) 21.3 -> 22.1, 256 21.1 -> 28.5;
// both products of a block of one, 5120 -> 2304 -> 5120: 64 rows 29.3 -> 21.3, 128 31.3 -> 29.1, 160 (108 and 120 tiles) 32.6 -> 40.1; two experts, 2048 x 2048, 300
// rows (96 tiles) 11.0 -> 10.9; where the tiles are more than run at once, 2304 -> 5120: 8 experts, 64 rows 39.7 -> 42.0; 48 experts, 384 rows 176 -> 184;
// six of them, 240 tiles, 29.1 -> 28.0.
// 8 bits, 5120 x 5120 of one weight: 16 rows 16.0 -> 8.6, 64 16.2 -> 12.7, 128 16.6 -> 16.2, 192 16.8 -> 24.6.  That line at 128 rows was drawn there; between 64 and it
// the weights are read for two tiles, which costs more the wider they are.  65 and 128 rows: 2304 -> 5120 10.3 -> 9.7, 10.4 -> 11.6; gated 5120 -> 2 x 2304 16.3 -> 13.8,
// 16.3 -> 15.4; gated 2048 -> 2 x 768 9.2 -> 6.8, 9.3 -> 7.4; 1024 -> 16384 10.5 -> 9.6, 10.9 -> 10.8; gated 5120 -> 2 x 8192 26.5 -> 27.7, 26.6 -> 31.7; 8192 -> 8192
// 24.1 -> 32.1, 24.1 -> 37.0; 8192 -> 16384 36.8 -> 40.3, 37.0 -> 46.1; gated 8192 -> 2 x 8192 37.3 -> 40.9, 37.7 -> 46.5.  More experts: a tile of few rows costs 560 clk a group of k and
// 6000, one of pairs (a half of it, which one SM has) 1026 and 2700.  16 experts, gated 1024 -> 2 x 512: 300 rows 11.1 -> 8.6.  48, gated 5120 -> 2 x 2304: 384
// rows 257 -> 188, 2304 271 -> 219, 2976 274 -> 239, 5000 285 -> 339.  48, 2304 -> 5120: 384 133 -> 112, 2304 140 -> 128, 3000 143 -> 145.  128, gated 2048 -> 2 x 768: 512
// 94 -> 77, 4096 104 -> 93, 8192 108 -> 121.  128, 768 -> 2048: 512 57 -> 60, 4096 64 -> 75.  Where all rows are one expert's pairs are ahead (48 experts, 3000 rows
// 75 -> 181, 8 experts, 500 rows 19 -> 33), which is not known here; where half of them are, not (323 -> 261, 52 -> 53).
bool grouped_few_rows(const GroupedProduct& p, int sms) {
  if (p.w_k_rows || (p.kind != kLinear && p.kind != kGated)) return false;
  if (p.type == kGroupedE4m3) {
    if (p.rows <= 128) return true;
    const int64_t each = (p.rows + p.experts - 1) / p.experts, groups = (p.k + kScaleBlock - 1) / kScaleBlock;
    if (each > kFewCols) return false;
    // an expert's rows come in each / 64 + 1/2 tiles on average, one at least
    return few_tiles(p) <= 2 * sms || std::max<int64_t>(kFewCols, each + kFewCols / 2) * (560 * groups + 6000) <= kFewCols * (1026 * groups + 2700);
  }
  return 3 * few_tiles(p) <= (p.rows <= kFewCols ? 6 : 2) * sms;
}

cudaError_t prepare_grouped_few() {
  return for_each_few_kernel([](auto kernel, bool, bool) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem); });
}

cudaError_t launch_grouped_few(const GroupedProduct& p, int sms, cudaStream_t s) {
  FewParams d = {};
  const bool fp8 = p.type == kGroupedE4m3, gate = p.kind == kGated;
  d.ends = p.ends, d.experts = p.experts, d.rows = p.rows, d.n = p.n;
  const int width = gate ? kFewRows / 2 : kFewRows;
  d.row_tiles = (p.n + width - 1) / width;
  d.k_stages = (p.k + (fp8 ? 127 : 63)) / (fp8 ? 128 : 64);
  d.blocks = (p.n + kScaleBlock - 1) / kScaleBlock;
  d.idesc = product_idesc(fp8 ? kDenseFp16 : p.type, false, false, kFewRows, 0);     // format 0: FP16, or in 8 bits E4M3
  d.tmem_cols = fp8 ? kFewAccumulators * kFewCols : kFewCols;
  d.x_scales = p.x_scales, d.w_scales = p.w_scales;
  d.epi = p.epi;
  d.zero_behind = p.zero_behind && p.ends != nullptr;
  d.status = p.status;
  d.timeout_ns = (p.timeout_ms > 0 ? (int64_t)p.timeout_ms : 2000) * 1000000ll;
  d.split = few_split(p, few_tiles(p), d.k_stages, sms);
  const uint64_t size = fp8 ? 1 : 2, n = p.n, k = p.k, parts = gate ? 2 : 1;
  const uint32_t depth = static_cast<uint32_t>(128 / size);
  bool ok = encode_map(&d.map_w, p.type, p.w, 4, {k, n, parts, static_cast<uint64_t>(p.experts), 1}, {k * size, n * k * size, parts * n * k * size, 0},
                       {depth, static_cast<uint32_t>(width), 1, 1, 1});
  for (int i = 0; ok && i < 3; ++i)
    ok = encode_map(&d.map_x[i], p.type, p.x, 2, {k, static_cast<uint64_t>(p.rows), 1, 1, 1}, {static_cast<uint64_t>(p.x_ld) * size, 0, 0, 0}, {depth, 64u >> i, 1, 1, 1});
  const int64_t most = ((int64_t)p.rows / kFewCols + std::min(p.experts, p.rows)) * d.row_tiles * d.split;
  if (!ok || most > INT32_MAX / 2) return cudaErrorInvalidValue;
  bool found = false;
  const cudaError_t e = for_each_few_kernel([&](auto kernel, bool k_fp8, bool k_gate) {
    if (k_fp8 != fp8 || k_gate != gate) return cudaSuccess;
    found = true;
    return launch_clustered(kernel, dim3(static_cast<uint32_t>(most)), dim3(kFewThreads), kFewSmem, d.split, s, d);
  });
  return found ? e : cudaErrorInvalidValue;
}

}  // namespace mmoe
