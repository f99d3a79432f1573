// Training forward pass of the GQA attention for sm_100a: O = softmax(s) V and
// each row's log-sum, s = q.k (scaled), on tcgen05 with TMEM accumulators.
//
// Items and pipeline are those of the backward kernel (attention_bwd.cu): a row
// item is 128 query rows (stationary Q) that walk the keys in chunks of 64, a
// persistent CTA per SM has all 512 columns of TMEM, one warp issues S = Q K^T of
// the next steps while the softmax of the current ones runs, another O += P V; four
// join the outputs and one stores them.
//
// Four sums per row. Two groups of compute warps take the steps in turn, and in
// a group two warps share each row, each with half of the chunk's keys. Each of
// these four streams is a softmax of its own over its quarter of the keys:
// running maximum, sum, and an accumulator of 64 columns, so that no warp waits
// for another's maximum. The streams are joined when the item ends:
//   m = max m_i,  L = sum 2^(m_i - m) l_i,  O = sum 2^(m_i - m) O_i / L.
// A stream's reference maximum only moves (and its O is rescaled in TMEM) when
// a chunk exceeds it by more than 8, a factor 256, as in the inference kernel.
//
// Long items of few heads are cut into parts, each a call's worth of streams of
// its own, whose O, m and L a second kernel joins, all in fp32 (the inference
// kernel's parts are held in bf16). P is rounded to bf16 as the operand of P V, or
// to twice that in fine calls (see kFineShare).
//
// Bound: no unit alone. A 128 x 64 step needs 512 cycles of the special-function
// units (its exponentials, 16 per cycle) and 368 of the products (4 SS of about 49
// and 4 TS of about 43, by their shared-memory reads and issue), and takes about
// 1000 (causal, 2 x 4096 rows, 15 heads: 214 steps per SM in 112 us): the chain from
// S in TMEM over the exponentials to P in TMEM, handed over by barriers at both
// ends, sets the time.
//
// Every mbarrier wait is bounded as in the inference kernel.

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "attention_common.cuh"
#include "attention_train.cuh"
#include "vlak_device.cuh"
#include "vlak_internal.h"

namespace vlak {
namespace {

constexpr int kRing = 6;                     // streamed (K, V) chunks in flight
constexpr int kTiles = 3;                    // items whose Q tile is in shared memory
constexpr int kStages = 4;                   // S tiles in TMEM
constexpr int kQueue = 8;                    // items handed out and not yet seen by every warp

constexpr int kGroupWarps = 8;               // as in the backward kernel
constexpr int kComputeWarps = 2 * kGroupWarps;
constexpr int kWarpProducer = kComputeWarps, kWarpScores = kComputeWarps + 1,
              kWarpAccum = kComputeWarps + 2;  // kComputeWarps + 3: stores
constexpr int kWarpOutput = kComputeWarps + 4, kOutputWarps = 4;
constexpr int kThreads = 32 * (kWarpOutput + kOutputWarps);
// Registers by warpgroup: compute, issue, output, whose four accumulators of 16
// columns are the most.
constexpr int kRegsLaunch = 80, kRegsCompute = 80, kRegsIssue = 40, kRegsOutput = 112;
static_assert(32 * kComputeWarps * kRegsCompute + 128 * kRegsIssue + 32 * kOutputWarps * kRegsOutput <=
                  kThreads * kRegsLaunch,
              "the split must fit the launch's registers");

// TMEM columns: the four streams' accumulators, then the stages; P (bf16 pairs)
// overwrites parts of S. Stream = 2 * group + half.
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kAcc = 0, kStage0 = 256, kStageCols = 64;
static_assert(kStage0 + kStages * kStageCols <= kTmemCols, "TMEM");
constexpr float kRescaleThreshold = 8.f;  // log2 units

struct __align__(64) FwdParams : TrainShape {
  CUtensorMap tm_q, tm_o;                    // dims (64, H, M, B), box (64, Gb, MT, 1)
  CUtensorMap tm_k, tm_v;                    // dims (64, Hkv, N, B), box (64, 1, 64, 1)
  float* lse;                                // (B, M, H), log2 units
  __nv_bfloat16* o;
  int8_t* o_low;                             // contiguous (B, M, H, 64), or null
  long long o_s[3];                          // (b, m, h) element strides
  int parts;                                 // of an item's steps; with several:
  float* sums;                               // [part][B * Hkv][n_sub * 64][64] O
  float2* ml;                                // [part][B * Hkv][n_sub * 64] m, L
  int n_items;                               // parts of all items
  FastDiv by_parts;
};

struct Barriers {
  uint64_t a_full[kTiles], a_empty[kTiles];  // Q tile of an item
  uint64_t b_full[kRing], b_empty[kRing];    // streamed chunks
  uint64_t s_full[kStages], x_full[kStages], t_empty[kStages];
  uint64_t pv_done[2];                       // [group]
  uint64_t ml_full[2], ml_empty[2];          // streams' maxima and sums of an item
  uint64_t out_full, staged[kTiles], acc_empty, drain[2];
  uint64_t it_full[kQueue], it_empty[kQueue];
  Item item[kQueue];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kBarrierBytes = 1024;
static_assert(sizeof(Barriers) <= kBarrierBytes, "barrier block");
constexpr int kTileBytes = 2 * kSubBytes;
constexpr int kMlFloats = 4 * 128 * 2;       // [stream][row] (m, l)
constexpr int kSmem = kTiles * kTileBytes + kRing * 2 * kSubBytes + 2 * kMlFloats * 4 + kBarrierBytes + 1024;
static_assert(kSmem <= 227 * 1024 && kSmem > 114 * 1024, "one CTA per SM");

template <int kMode>
__device__ __forceinline__ Item decode_item(const FwdParams& p, int id) {
  Item it{};
  const int i = fast_div(id, p.by_parts);
  const int outer = fast_div(i, p.bk_inner ? p.by_bk : p.by_pair);
  const int rest = i - outer * (p.bk_inner ? p.n_bk : p.n_pair);
  const int blk = p.bk_inner ? outer : rest, bk = p.bk_inner ? rest : outer;
  it.b = fast_div(bk, p.by_hkv);
  it.kvh = bk - it.b * p.Hkv;
  it.L = kMode == kMaskLength ? length_of(p, it.b) : 0;
  row_item<kMode>(p, blk, it);
  if (p.parts > 1) take_part(it, id - i * p.parts, p.parts);
  return it;
}

__device__ __forceinline__ void less_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
}

template <int kMode, bool kFine>
__global__ void __launch_bounds__(kThreads, 1) attn_train_fwd(const __grid_constant__ FwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* a_smem = smem;                           // [kTiles][Q 16 KB]; then the staged O
  uint8_t* b_smem = a_smem + kTiles * kTileBytes;   // [kRing][K 8 KB, V 8 KB]
  float2* ml_smem = reinterpret_cast<float2*>(b_smem + kRing * 2 * kSubBytes);  // [2][stream][row]
  Barriers* bars = reinterpret_cast<Barriers*>(ml_smem + kMlFloats);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(&bars->a_full[i], 1);
      mbar_init(&bars->a_empty[i], 1);
      mbar_init(&bars->staged[i], kOutputWarps);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bars->b_full[i], 1);
      mbar_init(&bars->b_empty[i], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->x_full[i], kGroupWarps);
      mbar_init(&bars->t_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->pv_done[i], 1);
      mbar_init(&bars->ml_full[i], kComputeWarps);
      mbar_init(&bars->ml_empty[i], kOutputWarps);
      mbar_init(&bars->drain[i], 1);
    }
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(&bars->it_full[i], 1);
      mbar_init(&bars->it_empty[i], kComputeWarps + 3 + kOutputWarps);
    }
    mbar_init(&bars->out_full, 1);
    mbar_init(&bars->acc_empty, kOutputWarps);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpAccum) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // an allocation of all 512 columns starts at the first; as a constant, it keeps
  // the issue warps' operands uniform
  constexpr uint32_t tmem = 0;

  auto take_item = [&](uint32_t n, Item& it) {
    const uint32_t q = n % kQueue;
    if (!__all_sync(kFullMask, bounded_wait<1>(&bars->it_full[q], (n / kQueue) & 1, abort_flag)))
      return false;
    it = load_item(&bars->item[q]);
    __syncwarp();
    mbar_arrive_elect(&bars->it_empty[q]);
    return true;
  };

  if (warp == kWarpProducer) {
    less_registers();
    uint32_t t = 0, live = 0;  // steps and live items issued
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t q = n % kQueue;
      if (!__all_sync(kFullMask, bounded_wait(&bars->it_empty[q], ((n / kQueue) & 1) ^ 1, abort_flag)))
        break;
      // items in turn over the CTAs. Under a staircase the long ones come first, so
      // every other round goes in reverse, else the first CTA had the longest of
      // each: causal, 2 x 4096 rows, 15 / 5 heads, 125 -> 116 us
      const bool back = kMode == kMaskAnalytic && (n & 1);
      const long long id =
          static_cast<long long>(n) * gridDim.x + (back ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      Item it{};
      if (id < p.n_items)
        it = decode_item<kMode>(p, static_cast<int>(id));
      else
        it.live = -1;
      if (lane == 0) {
        bars->item[q] = it;
        mbar_arrive(&bars->it_full[q]);
      }
      __syncwarp();
      if (it.live < 0) break;
      if (it.live == 0) continue;
      const uint32_t ab = live % kTiles;
      if (!__all_sync(kFullMask, bounded_wait(&bars->a_empty[ab], ((live / kTiles) & 1) ^ 1, abort_flag)))
        break;
      mbar_arrive_expect_tx_elect(&bars->a_full[ab],
                                  static_cast<uint32_t>(it.n_here * p.Gb * p.MT * kRowBytes));
      for (int i = 0; i < it.n_here; ++i) {
        const int hb = fast_div(it.s0 + i, p.by_mt_count), m0 = (it.s0 + i - hb * p.n_mt) * p.MT;
        tma_load_4d_elect(a_smem + ab * kTileBytes + i * kSubBytes, &p.tm_q, &bars->a_full[ab], 0,
                          it.kvh * p.G + hb * p.Gb, m0, it.b);
      }
      ++live;
      Steps step;
      step.begin(it);
      for (int j = 0; j < it.live; ++j, ++t, step.next(it)) {
        const uint32_t s = t % kRing;
        if (!__all_sync(kFullMask, bounded_wait(&bars->b_empty[s], ((t / kRing) & 1) ^ 1, abort_flag))) {
          ok = false;
          break;
        }
        uint8_t* b0 = b_smem + s * 2 * kSubBytes;
        mbar_arrive_expect_tx_elect(&bars->b_full[s], 2 * kSubBytes);
        tma_load_4d_elect(b0, &p.tm_k, &bars->b_full[s], 0, it.kvh, step.pos * kChunk, it.b);
        tma_load_4d_elect(b0 + kSubBytes, &p.tm_v, &bars->b_full[s], 0, it.kvh, step.pos * kChunk, it.b);
      }
    }
    // never leave the CTA with copies in flight (bounded, abort or not)
    for (uint32_t k = live > kTiles ? live - kTiles : 0; k < live; ++k)
      bounded_wait(&bars->a_full[k % kTiles], (k / kTiles) & 1, abort_flag, false);
    for (uint32_t k = t > kRing ? t - kRing : 0; k < t; ++k)
      bounded_wait(&bars->b_full[k % kRing], (k / kRing) & 1, abort_flag, false);
    __syncwarp();
  } else if (warp == kWarpScores) {
    less_registers();
    // S = Q K^T of every step, up to kStages steps ahead of the products with V.
    // Its waits suspend the warp, unlike the others': 4 x 1024 rows, 12 heads 30.4 ->
    // 29.3 us (all of them suspended 29.7, the backward kernel's 59.5 -> 62).
    const uint32_t id_kk = idesc_bf16_f32(128, 64, false);
    const uint64_t a_desc = sdesc_sw128(smem_u32(a_smem)), b_desc = sdesc_sw128(smem_u32(b_smem));
    // V rows that no query sees meet P = 0 only, and may hold NaN: cleared
    const bool dead = kMode == kMaskLength || (kMode == kMaskAnalytic && p.ds < p.de);
    Turn<kTiles> ab;
    Turn<kRing> s;
    Turn<kStages> st;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      if (!__all_sync(kFullMask, bounded_wait(&bars->a_full[ab.i], ab.round, abort_flag))) break;
      const uint64_t a0 = a_desc + ab.i * (kTileBytes / 16);
      ab.next();
      Steps step;
      step.begin(it);
      for (int j = 0; j < it.live; ++j) {
        if (!__all_sync(kFullMask, bounded_wait(&bars->t_empty[st.i], st.round ^ 1, abort_flag) &&
                                       bounded_wait(&bars->b_full[s.i], s.round, abort_flag))) {
          ok = false;
          break;
        }
        if (dead) {
          const int c0 = step.pos * kChunk;
          const int lo = kMode == kMaskLength ? it.L - c0 : p.ds - c0;
          const int hi = kMode == kMaskLength ? kChunk : p.de - c0;
          clear_rows(b_smem + s.i * 2 * kSubBytes + kSubBytes, max(lo, 0), min(hi, kChunk));
          step.next(it);
        }
        tc_fence_after();
        umma_ss_x4(tmem + kStage0 + st.i * kStageCols, a0, b_desc + s.i * (2 * kSubBytes / 16), id_kk);
        umma_commit_elect(&bars->s_full[st.i]);
        s.next();
        st.next();
      }
    }
    // every issued product completes before TMEM is released
    umma_commit_elect(&bars->drain[0]);
    bounded_wait(&bars->drain[0], 0, abort_flag, false);
    __syncwarp();
  } else if (warp == kWarpAccum) {
    less_registers();
    // Both halves' accumulators of the step's group += P V, 32 keys each.
    const uint32_t id_kn = idesc_bf16_f32(128, 64, true);
    const uint64_t v_desc = sdesc_sw128(smem_u32(b_smem)) + kSubBytes / 16;
    Turn<kRing> s;
    Turn<kStages> st;
    uint32_t t = 0, live = 0;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      // the previous item's accumulators have been read
      if (live > 0 &&
          !__all_sync(kFullMask, bounded_wait<1>(&bars->acc_empty, (live - 1) & 1, abort_flag)))
        break;
      for (int j = 0; j < it.live; ++j, ++t) {
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->x_full[st.i], st.round, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t x = tmem + kStage0 + st.i * kStageCols, d = tmem + kAcc + (t & 1) * 128;
        const uint64_t v0 = v_desc + s.i * (2 * kSubBytes / 16);
        umma_ts_x2(d, x, v0, id_kn, j > 1);
        umma_ts_x2(d + 64, x + 32, v0 + 256, id_kn, j > 1);
        if (kFine) {  // the rests of P
          umma_ts_x2(d, x + 16, v0, id_kn, 1u);
          umma_ts_x2(d + 64, x + 48, v0 + 256, id_kn, 1u);
        }
        umma_commit_elect(&bars->pv_done[t & 1]);
        umma_commit_elect(&bars->t_empty[st.i]);
        umma_commit_elect(&bars->b_empty[s.i]);
        s.next();
        st.next();
      }
      if (!ok) break;
      umma_commit_elect(&bars->out_full);
      ++live;
    }
    umma_commit_elect(&bars->drain[1]);
    bounded_wait(&bars->drain[1], 0, abort_flag, false);
    __syncwarp();
  } else if (warp < kComputeWarps) {
    static_assert(kRegsCompute == kRegsLaunch, "compute warps keep the launch's registers");
    // Compute warps: a row per lane, 32 of a step's 64 keys; the softmax of one
    // stream.
    const int group = warp >> 3, quarter = warp & 3, gq = (warp >> 2) & 1;
    const int tl = quarter * 32 + lane;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_acc = tbase + kAcc + (2 * group + gq) * 64;
    const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
    uint32_t t = 0, live = 0, mine = 0;  // steps, live items, steps of the group
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      const SubRow r = sub_row(p, it.s0 + (quarter >> 1), (quarter & 1) * 32 + lane);
      // keys [0, from) and [mid, to) are seen by the row
      int from = 0, mid = 0, to = 0;
      if (kMode == kMaskAnalytic) {
        from = p.ds;
        mid = p.de;
        to = max(p.P, min(p.N, p.N - p.M + r.m + 1));
      } else if (kMode == kMaskLength) {
        to = r.m < it.L ? it.L : 0;
      }
      constexpr int kFar = INT32_MAX / 2;
      const int to_lo = __reduce_min_sync(kFullMask, r.valid ? to : kFar);
      const int to_hi = __reduce_max_sync(kFullMask, r.valid ? to : -kFar);
      float m_run = -INFINITY, l_run = 0.f;
      // this group's steps: every other one
      const int j0 = static_cast<int>((t ^ group) & 1u);
      for (int j = j0; j < it.live; j += 2, ++mine) {
        const int k = it.j0 + j;
        const int c = (k < it.a1 ? k : k - it.a1 + it.b0) * kChunk + 32 * gq;
        // which of the 32 keys this row sees; all or none for the whole warp
        // (lanes without a row do not count)
        uint32_t vm = 0u;
        bool full, none;
        if (kMode == kMaskBool) {
          if (r.valid && c < p.N) vm = row_bits_at(p, it.b, r.m, c);
          full = __all_sync(kFullMask, !r.valid || vm == 0xffffffffu);
          none = __all_sync(kFullMask, !r.valid || vm == 0u);
        } else {
          full = c + 32 <= from || (c >= mid && c + 32 <= to_lo);
          none = c >= from && (c + 32 <= mid || c >= to_hi);
          if (!full && !none) vm = low_bits(from - c) | (low_bits(to - c) & ~low_bits(mid - c));
        }
        const uint32_t tj = t + j, st = tj % kStages;
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->s_full[st], (tj / kStages) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t0 = tbase + kStage0 + st * kStageCols + 32 * gq;
        if (none) {
          const uint32_t zero[16] = {};
          tmem_st16(t0, zero);
          if (kFine) tmem_st16(t0 + 16, zero);
        } else {
          float sv[32];
          tmem_ld32(t0, sv);
          tmem_wait_ld();
          if (!full) {
#pragma unroll
            for (int i = 0; i < 32; ++i) sv[i] = (vm >> i) & 1u ? sv[i] : -INFINITY;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], sv[i], sv[i + 1]);
          const float mz = fmax3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * p.scale_log2;
          float alpha = 1.f;
          if (m_run == -INFINITY) {
            m_run = mz;  // the sum and the accumulator are still zero
          } else if (mz > m_run + kRescaleThreshold) {
            alpha = ex2(m_run - mz);
            m_run = mz;
          }
          const float nref = m_run == -INFINITY ? 0.f : -m_run;
          const uint64_t nr2 = f2_pack(nref, nref);
          uint64_t acc[2] = {0ull, 0ull};
          uint32_t pk[16], rest[4];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(sv[2 * i], sv[2 * i + 1]), sl2, nr2), x0, x1);
            const float e0 = ex2(x0), e1 = ex2(x1);
            acc[i & 1] = f2_add(acc[i & 1], f2_pack(e0, e1));
            pk[i] = pack_bf16x2(e0, e1);
            if (kFine) {
              rest[i % 4] = rest_of_pair(e0, e1, pk[i]);
              if (i % 4 == 3) {
                tmem_st4(t0 + i - 3, pk + i - 3);
                tmem_st4(t0 + 16 + i - 3, rest);
              }
            }
          }
          if (!kFine) tmem_st16(t0, pk);
          float a0, a1;
          f2_unpack(f2_add(acc[0], acc[1]), a0, a1);
          l_run = l_run * alpha + (a0 + a1);
          // Rare: the reference moved. The stream's products so far are rescaled
          // once they are done (only in the item's later steps are there any).
          if (j > 1 && __any_sync(kFullMask, alpha != 1.f)) {
            if (!__all_sync(kFullMask, bounded_wait(&bars->pv_done[group], (mine - 1) & 1, abort_flag))) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              float o[16];
              tmem_ld16(t_acc + 16 * q, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16f(t_acc + 16 * q, o);
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_elect(&bars->x_full[st]);
      }
      if (!ok) break;
      // the stream's maximum and sum, for the output warps
      const uint32_t mb = live & 1;
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->ml_empty[mb], ((live >> 1) & 1) ^ 1, abort_flag))) break;
      ml_smem[(mb * 4 + 2 * group + gq) * 128 + tl] = make_float2(m_run, l_run);
      __syncwarp();
      mbar_arrive_elect(&bars->ml_full[mb]);
      t += it.live;
      ++live;
    }
  } else if (warp >= kWarpOutput) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsOutput));
    // Outputs: the streams joined, staged over the item's Q tile in the swizzled
    // layout of the map; or a part's sums. One lane quarter of
    // TMEM per warp.
    const int quarter = warp & 3;
    const int tl = quarter * 32 + lane;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t t = 0, live = 0;
    Turn<kTiles> ab;
    for (uint32_t n = 0;; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      const SubRow r = sub_row(p, it.s0 + (quarter >> 1), (quarter & 1) * 32 + lane);
      const int h = it.kvh * p.G + r.g;
      const long long row = (static_cast<long long>(it.b) * p.M + r.m) * p.H + h;
      long long part_row = 0;
      if (p.parts > 1)
        part_row = (static_cast<long long>(it.part) * p.n_bk + it.b * p.Hkv + it.kvh) * p.n_sub * kSub +
                   static_cast<long long>(it.s0) * kSub + tl;
      if (it.live == 0) {  // no key seen
        if (p.parts > 1) {
          if (r.valid) p.ml[part_row] = make_float2(-INFINITY, 0.f);
        } else if (r.valid) {
          uint4* dst = reinterpret_cast<uint4*>(p.o + it.b * p.o_s[0] + r.m * p.o_s[1] + h * p.o_s[2]);
#pragma unroll
          for (int v = 0; v < 8; ++v) dst[v] = make_uint4(0, 0, 0, 0);
          p.lse[row] = -INFINITY;
        }
        continue;
      }
      // weights of the streams; those of a group without steps have none
      const uint32_t mb = live & 1;
      const bool has[2] = {it.live > 1 || (t & 1) == 0, it.live > 1 || (t & 1) == 1};
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->ml_full[mb], (live >> 1) & 1, abort_flag))) break;
      float w[4], m = -INFINITY, L = 0.f;
      {
        float2 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = ml_smem[(mb * 4 + i) * 128 + tl];
          m = fmaxf(m, x[i].x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = x[i].y == 0.f ? 0.f : ex2(x[i].x - m);
          L += w[i] * x[i].y;
        }
      }
      __syncwarp();
      mbar_arrive_elect(&bars->ml_empty[mb]);
      const float inv = L == 0.f ? 0.f : __fdividef(1.f, L);
      if (p.parts > 1) {
        if (r.valid) p.ml[part_row] = make_float2(m, L);
      } else {
        if (r.valid) p.lse[row] = L == 0.f ? -INFINITY : m + __log2f(L);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] *= inv;
      }
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->out_full, live & 1, abort_flag))) break;
      tc_fence_after();
      uint8_t* a0 = a_smem + ab.i * kTileBytes;
      float* sums = p.parts > 1 ? p.sums + part_row * 64 : nullptr;
      uint8_t* stage = a0 + tl * kRowBytes;
      uint4* low = p.parts == 1 && p.o_low != nullptr && r.valid ? reinterpret_cast<uint4*>(p.o_low + row * 64)
                                                                 : nullptr;
      uint64_t w2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w2[i] = f2_pack(w[i], w[i]);
#pragma unroll 1
      for (int q = 0; q < 4; ++q) {  // 16 columns of the four streams at a time
        float x[4][16];
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (has[g]) {
            tmem_ld16(tbase + kAcc + 128 * g + 16 * q, x[2 * g]);
            tmem_ld16(tbase + kAcc + 128 * g + 64 + 16 * q, x[2 * g + 1]);
          }
        tmem_wait_ld();
        if (q == 3) {  // read: the next item may accumulate
          tc_fence_before();
          mbar_arrive_elect(&bars->acc_empty);
        }
        uint64_t o2[8] = {};
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if (has[g]) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o2[i] = f2_fma(f2_pack(x[2 * g + 1][2 * i], x[2 * g + 1][2 * i + 1]), w2[2 * g + 1],
                             f2_fma(f2_pack(x[2 * g][2 * i], x[2 * g][2 * i + 1]), w2[2 * g], o2[i]));
          }
        float o[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) f2_unpack(o2[i], o[2 * i], o[2 * i + 1]);
        if (p.parts > 1) {
          if (r.valid) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              reinterpret_cast<float4*>(sums)[4 * q + v] =
                  make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        } else {
          uint32_t hi[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) hi[i] = L == 0.f ? 0u : pack_bf16x2(o[2 * i], o[2 * i + 1]);
#pragma unroll
          for (int v = 0; v < 2; ++v)
            st_shared_v4(stage + (static_cast<uint32_t>(2 * q + v) ^ static_cast<uint32_t>(tl & 7)) * 16,
                         hi[4 * v], hi[4 * v + 1], hi[4 * v + 2], hi[4 * v + 3]);
          if (low != nullptr)
            low[q] = make_uint4(low_bytes(o, hi), low_bytes(o + 4, hi + 2), low_bytes(o + 8, hi + 4),
                                low_bytes(o + 12, hi + 6));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(&bars->staged[ab.i]);
      ab.next();
      t += it.live;
      ++live;
    }
  } else {
    less_registers();
    // Stores of the staged outputs, which release the items' tiles. (In the output
    // warps they took 2 to 3K cycles of an item's 7K.) A tile's barrier is not
    // arrived at again before the tile has been released.
    Turn<kTiles> ab;
    for (uint32_t n = 0;; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->staged[ab.i], ab.round, abort_flag))) break;
      if (lane == 0) {
        if (p.parts == 1) {
          for (int i = 0; i < it.n_here; ++i) {
            const int hb = fast_div(it.s0 + i, p.by_mt_count), m0 = (it.s0 + i - hb * p.n_mt) * p.MT;
            tma_store_4d(&p.tm_o, a_smem + ab.i * kTileBytes + i * kSubBytes, 0, it.kvh * p.G + hb * p.Gb, m0,
                         it.b);
          }
          bulk_commit_group();
          bulk_wait_read0();
        }
        mbar_arrive(&bars->a_empty[ab.i]);
      }
      __syncwarp();
      ab.next();
    }
    // the stores complete before the CTA exits
    if (lane == 0) bulk_wait_all0();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) publish_device_error(p.host_err, VLAK_ERR_DEVICE_TIMEOUT);
  if (warp == kWarpAccum) {
    tc_fence_after();
    tmem_dealloc(bars->tmem_base, kTmemCols);
  }
}

// Joins the parts of each row, in their order: blockIdx.y (b, kv head),
// blockIdx.x a quarter of a sub-tile, 16 threads of four columns per row.
__global__ void __launch_bounds__(256) attn_train_fwd_join(const __grid_constant__ FwdParams p) {
  const int st = blockIdx.x >> 2, row64 = (blockIdx.x & 3) * 16 + (threadIdx.x >> 4);
  const int bk = blockIdx.y, v = threadIdx.x & 15;
  const SubRow r = sub_row(p, st, row64);
  if (!r.valid) return;
  const long long rows = static_cast<long long>(p.n_sub) * kSub, stride = p.n_bk * rows;
  const long long at = bk * rows + static_cast<long long>(st) * kSub + row64;
  float m = -INFINITY;
  for (int k = 0; k < p.parts; ++k) m = fmaxf(m, p.ml[k * stride + at].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float L = 0.f;
#pragma unroll 4
  for (int k = 0; k < p.parts; ++k) {
    const float2 ml = p.ml[k * stride + at];
    if (ml.y == 0.f) continue;  // saw no key: its sums were not written
    const float w = ex2(ml.x - m);
    const float4 x = reinterpret_cast<const float4*>(p.sums + (k * stride + at) * 64)[v];
    L += w * ml.y;
    o.x += w * x.x;
    o.y += w * x.y;
    o.z += w * x.z;
    o.w += w * x.w;
  }
  const int b = fast_div(bk, p.by_hkv), kvh = bk - b * p.Hkv, h = kvh * p.G + r.g;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const long long row = (static_cast<long long>(b) * p.M + r.m) * p.H + h;
  const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  const uint32_t hi[2] = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
  *reinterpret_cast<uint2*>(p.o + b * p.o_s[0] + r.m * p.o_s[1] + h * p.o_s[2] + 4 * v) =
      make_uint2(hi[0], hi[1]);
  if (p.o_low != nullptr) *reinterpret_cast<uint32_t*>(p.o_low + row * 64 + 4 * v) = low_bytes(x, hi);
  if (v == 0)
    p.lse[row] = L == 0.f ? -INFINITY : m + log2f(L);
}

// N == 0: zeros, and log-sums of -inf.
__global__ void no_keys(__nv_bfloat16* o, long long o_sb, long long o_sm, long long o_sh, float* lse, int M,
                        int H, long long rows) {
  for (long long r = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; r < rows;
       r += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long h = r % H, bm = r / H, m = bm % M, b = bm / M;
    uint4* dst = reinterpret_cast<uint4*>(o + b * o_sb + m * o_sm + h * o_sh);
#pragma unroll
    for (int v = 0; v < 8; ++v) dst[v] = make_uint4(0, 0, 0, 0);
    lse[r] = -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// host

// Parts and workspace of a call: the parts' sums, their maxima and sums, and the
// packed mask.
struct FwdPlan {
  SubTiling tl;
  int64_t n_bk, n_pair;
  int parts;
  bool fine;
  int64_t ml, bits, bytes;
};
FwdPlan plan_fwd(const vlak_attn_gqa_args* a, bool masked) {
  FwdPlan w{};
  w.tl = sub_tiling(static_cast<int>(a->H / a->Hkv), static_cast<int>(a->M));
  w.n_bk = a->B * a->Hkv;
  w.n_pair = (w.tl.n_sub + 1) / 2;
  const int64_t n_chunks = (a->N + kChunk - 1) / kChunk;
  const int64_t total = w.n_bk * w.n_pair * n_chunks;
  w.parts = item_parts(n_chunks, total);
  w.fine = fine_call(*a, total);
  if (w.parts > 1) {
    const int64_t rows = w.parts * w.n_bk * w.tl.n_sub * kSub;
    w.ml = rows * 64 * 4;
    w.bits = w.ml + rows * 8;
  }
  w.bytes = w.bits + (masked ? row_bits_bytes(*a) : 0);
  return w;
}

template <int kMode, bool kFine>
cudaError_t launch_fwd(const FwdParams& p, unsigned grid, cudaStream_t cs, int device) {
  static std::atomic<int> ready[64];
  if (ready[device].load() == 0) {
    const cudaError_t e = cudaFuncSetAttribute(attn_train_fwd<kMode, kFine>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    ready[device].store(1);
  }
  attn_train_fwd<kMode, kFine><<<grid, kThreads, kSmem, cs>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || p.parts == 1) return e;
  attn_train_fwd_join<<<dim3(p.n_sub * 4, p.n_bk), 256, 0, cs>>>(p);
  return cudaGetLastError();
}

int run_fwd(const vlak_attn_train_args* t, void* workspace, int64_t ws_bytes, void* stream) {
  clear_error();
  const char* op = "fused_attention_gqa_train";
  vlak_attn_train_args args{};
  if (!t) return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null arguments", op);
  args = *t;
  if (args.lengths || args.mask) {
    args.attn.prefix_len = -1;
    args.attn.dead_start = args.attn.dead_end = 0;
  }
  const vlak_attn_gqa_args* a = &args.attn;
  int64_t P = 0;
  float scale = 0.f;
  int st = check_train(a, &P, &scale, op);
  if (st == VLAK_OK) st = check_train_masks(args, op);
  if (st != VLAK_OK) return st;
  if (reinterpret_cast<uintptr_t>(args.lse) % 4 != 0)
    return set_errorf(VLAK_ERR_ALIGNMENT, "%s: lse must be 4-byte aligned", op);
  const int64_t rows = a->B * a->M * a->H;
  if (rows == 0) return VLAK_OK;
  if (reinterpret_cast<uintptr_t>(args.o_low) % 16 != 0)
    return set_errorf(VLAK_ERR_ALIGNMENT, "%s: o_low must be 16-byte aligned", op);
  if (!a->o || !args.lse || (a->N > 0 && (!a->q || !a->k || !a->v)))
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", op);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const FwdPlan plan = plan_fwd(a, args.mask != nullptr);
  if (a->N > 0 && plan.bytes > 0 && (!workspace || ws_bytes < plan.bytes))
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: workspace missing or too small", op);
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return set_errorf(VLAK_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", op);
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != VLAK_OK) return st;
  if (dev.cc_major != 10)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DEVICE, "%s: needs an sm_100 device (found sm_%d%d)", op,
                      dev.cc_major, dev.cc_minor);
  if (dev.device >= 64) return set_error(VLAK_ERR_CUDA, "device ordinal out of range");
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a->o);
  if (a->N == 0) {
    no_keys<<<static_cast<int>(std::min<int64_t>((rows + 255) / 256, 4096)), 256, 0, cs>>>(
        o, a->o_stride[0], a->o_stride[1], a->o_stride[2], args.lse, static_cast<int>(a->M),
        static_cast<int>(a->H), rows);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? VLAK_OK : set_cuda_error(op, e);
  }
  const int64_t n_items = plan.n_bk * plan.n_pair * plan.parts;
  if (n_items > INT32_MAX || plan.n_bk * plan.tl.n_sub > INT32_MAX)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: too many work items", op);

  FwdParams p;
  memset(&p, 0, sizeof(p));
  static_cast<TrainShape&>(p) = train_shape(a, P, scale, plan.tl);
  set_masks(p, args);
  p.host_err = host_error_word(cs);
  p.lse = args.lse;
  p.o = o;
  p.o_low = static_cast<int8_t*>(args.o_low);
  for (int d = 0; d < 3; ++d) p.o_s[d] = a->o_stride[d];
  p.parts = plan.parts;
  p.sums = static_cast<float*>(workspace);
  p.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.ml);
  p.row_bits = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + plan.bits);
  p.n_items = static_cast<int>(n_items);
  p.by_parts = fast_div_by(static_cast<unsigned>(p.parts));
  const uint32_t gb = static_cast<uint32_t>(plan.tl.Gb), mt = static_cast<uint32_t>(plan.tl.MT);
  st = encode_map(&p.tm_q, a->q, a->H, a->M, a->B, a->q_stride[2], a->q_stride[1], a->q_stride[0], gb, mt, "q");
  if (st == VLAK_OK)
    st = encode_map(&p.tm_o, a->o, a->H, a->M, a->B, a->o_stride[2], a->o_stride[1], a->o_stride[0], gb, mt, "o");
  if (st == VLAK_OK)
    st = encode_map(&p.tm_k, a->k, a->Hkv, a->N, a->B, a->k_stride[2], a->k_stride[1], a->k_stride[0], 1,
                    kChunk, "k");
  if (st == VLAK_OK)
    st = encode_map(&p.tm_v, a->v, a->Hkv, a->N, a->B, a->v_stride[2], a->v_stride[1], a->v_stride[0], 1,
                    kChunk, "v");
  if (st != VLAK_OK) return st;
  const unsigned grid = static_cast<unsigned>(std::min(p.n_items, dev.sm_count));
  cudaError_t e = args.mask ? launch_pack(args, p, cs) : cudaSuccess;
  auto launch = [&](auto fine) {
    constexpr bool kFine = decltype(fine)::value;
    return args.lengths ? launch_fwd<kMaskLength, kFine>(p, grid, cs, dev.device)
           : args.mask  ? launch_fwd<kMaskBool, kFine>(p, grid, cs, dev.device)
                        : launch_fwd<kMaskAnalytic, kFine>(p, grid, cs, dev.device);
  };
  if (e == cudaSuccess) e = plan.fine ? launch(std::true_type()) : launch(std::false_type());
  return e == cudaSuccess ? VLAK_OK : set_cuda_error("fused_attention_gqa_train launch failed", e);
}

}  // namespace

int take_train_fwd_device_error(int* code) { return take_device_error(code); }

}  // namespace vlak

extern "C" int vlak_attn_gqa_train_fwd(const vlak_attn_train_args* args, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  return vlak::run_fwd(args, workspace, workspace_bytes, stream);
}

extern "C" int vlak_attn_gqa_train_workspace_size(const vlak_attn_train_args* args, int64_t* bytes) {
  using namespace vlak;
  clear_error();
  if (!bytes) return set_error(VLAK_ERR_INVALID_ARGUMENT, "workspace size: null output");
  *bytes = 0;
  if (!args) return set_error(VLAK_ERR_INVALID_ARGUMENT, "workspace size: null arguments");
  vlak_attn_gqa_args a = args->attn;
  if (args->lengths || args->mask) {
    a.prefix_len = -1;
    a.dead_start = a.dead_end = 0;
  }
  const int st = check_train(&a, nullptr, nullptr, "workspace size");
  if (st != VLAK_OK) return st;
  if (a.B > 0 && a.M > 0 && a.N > 0) *bytes = plan_fwd(&a, args->mask != nullptr).bytes;
  return VLAK_OK;
}
