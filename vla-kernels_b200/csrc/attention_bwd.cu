// Backward pass of the GQA attention (attention_gqa.cu) for sm_100a: tcgen05
// products with TMEM accumulators, probabilities recomputed from the scores.
//
// Mathematics, per query head with s = q.k (scaled), P = exp(s - logsumexp):
//   dV = P^T dO,  dP = dO V^T,  D = rowsum(dO * O),  dS = P * (dP - D),
//   dQ = scale dS K,  dK = scale dS^T Q,
// dK and dV summed over the G query heads of a kv head. Scores are taken in
// the exp2 domain: P = 2^(scale log2(e) s - lse), lse from the forward pass.
//
// A first small kernel (attn_bwd_stats) computes D and lays (-lse, -D) out by
// sub-tiles. The second, persistent, one works through two kinds of items that
// share no sums, so without atomics on results, which repeat bit for bit:
//   dkv  128 keys of a kv head, stationary K and V; walks the query rows of all
//        G heads: S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO, dK += dS^T Q
//        with P^T and dS^T as TMEM operands (keys along the lanes, so nothing is
//        transposed through shared memory);
//   dq   128 query rows, stationary Q and dO; walks the keys: S = Q K^T,
//        dP = dO V^T, then dQ += dS K with dS as a TMEM operand.
// Both are one loop: two stationary tiles A0, A1 (128 x 64), a stream of pairs
// B0, B1 (64 x 64), T0 = A0 B0^T and T1 = A1 B1^T, elementwise X1 = dS (and
// X0 = P), acc1 += X1 B0 (and acc0 += X0 B1). Scores and dP are computed in both
// (7 products instead of 5): joining dQ across key blocks would take atomics or
// a pass over partial sums.
//
// Pipeline. One CTA per SM with all 512 columns of TMEM: two accumulators and
// three stages of (T0, T1), so the products of the next steps, also those of the
// next item, are issued while the current one's elementwise part runs. Sixteen
// compute warps in two groups take the steps in turn, one warp issues the score
// products and another the accumulating ones, four carry the outputs away and one
// stores them. Items come from a counter, the long ones first; long items of few
// heads are cut into parts, whose fp32 sums another kernel joins in their order.
//
// Bound: by the products' shared-memory reads and issue. A step (128 x 64) is
// 8 SS products of about 49 cycles and 4 (dq) or 8 (dkv) TS products of about 43.
//
// Rounding: P and dS are rounded to bf16 as operands of the second products, as
// the forward pass rounds P, or to twice that in fine calls (see kFineShare);
// all sums, D and the statistics are fp32.
//
// Rows are cut into sub-tiles as attention_train.cuh says: two are the 128 rows
// of a dq item, one is the 64 columns of a dkv step.
//
// Every mbarrier wait is bounded as in the forward kernel.

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

constexpr int kKeys = 128;                   // keys of a dkv item
constexpr int kRing = 6;                     // streamed pairs in flight (even: see the compute warps' waits)
constexpr int kTiles = 3;                    // items whose stationary tiles are in shared memory
constexpr int kStages = 3;                   // (T0, T1) pairs in TMEM
constexpr int kQueue = 8;                    // items handed out and not yet seen by every warp
constexpr int kStatFloats = 2 * kSub;        // -lse and -D of a sub-tile
constexpr int kStatBytes = kStatFloats * 4;

// Compute warps: two groups of eight that take the steps in turn; of a group,
// two warps per lane quarter of TMEM, each with half of a step's 64 columns.
constexpr int kGroupWarps = 8;
constexpr int kComputeWarps = 2 * kGroupWarps;
// One warp issues the scores, another the accumulating products: one alone
// took about 1.6K cycles per step for both, three times the products' own time.
// Four more, one per lane quarter, carry the outputs away, so that no compute
// group pauses at an item's end (an item of three steps took twice as long
// when the groups did it in turn).
constexpr int kWarpProducer = kComputeWarps, kWarpScores = kComputeWarps + 1,
              kWarpAccum = kComputeWarps + 2;  // kComputeWarps + 3: stores
constexpr int kWarpOutput = kComputeWarps + 4, kOutputWarps = 4;
constexpr int kThreads = 32 * (kWarpOutput + kOutputWarps);
// Registers: a compute thread wants more than an even share, the others less.
constexpr int kRegsLaunch = 80, kRegsCompute = 88, kRegsOther = 64;
static_assert(32 * kComputeWarps * kRegsCompute + (kThreads - 32 * kComputeWarps) * kRegsOther <=
                  kThreads * kRegsLaunch,
              "the split must fit the launch's registers");

// TMEM columns: accumulators, then the stages; X0 and X1 (bf16 pairs) overwrite
// parts of T0 and T1
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kAcc0 = 0, kAcc1 = 64, kStage0 = 128, kStageCols = 128, kT1 = 64;
static_assert(kStage0 + kStages * kStageCols <= kTmemCols, "TMEM");

struct __align__(64) BwdParams : TrainShape {
  CUtensorMap tm_q, tm_do, tm_dq;            // dims (64, H, M, B), box (64, Gb, MT, 1)
  CUtensorMap tm_k64, tm_v64;                // dims (64, Hkv, N, B), box (64, 1, 64, 1)
  CUtensorMap tm_k, tm_v, tm_dk, tm_dv;      // the same, box (64, 1, 128, 1)
  __nv_bfloat16 *dq, *dk, *dv;               // contiguous
  const __nv_bfloat16 *o, *d_o;
  const int8_t* o_low;                       // contiguous (B, M, H, 64), or null
  long long o_s[3], do_s[3];                 // (b, m, h) element strides
  const float* lse;                          // (B, M, H), log2 units
  float* stats;                              // [B * Hkv][n_sub][-lse 64, -D 64]
  // Parts of a dkv and of a dq item's steps; with several, each leaves its sums
  // in fp32: [part][item][128 keys][dK 64, dV 64] and [part][sub-tile][64][64].
  int kv_parts, q_parts;
  float *kv_sums, *q_sums;
  int n_kblk, n_dkv, n_items;                // dkv parts; all parts
  float out_scale;
  FastDiv by_kblk, by_kv_parts, by_q_parts;
};

// Softmax over a single key is constant: its score's gradient is exactly zero. So
// where no row sees more keys, dQ and dK are scaled by zero: in the whole call
// (out_scale; see run_bwd), or in a sample of length 1.
__device__ __forceinline__ float scale_of(const BwdParams& p, int L) { return L == 1 ? 0.f : p.out_scale; }

// ---------------------------------------------------------------------------
// D = rowsum(dO * O), O with its low bytes, and -lse by sub-tile rows: four
// threads per row, two 16-byte vectors of each tensor per thread. Rows that do not
// exist or see no key get -lse = -inf (every P is 0) and D = 0, whatever memory
// holds there. Bound: HBM, one read of O and dO.
constexpr int kStatThreads = 4 * kSub;
__global__ void __launch_bounds__(kStatThreads) attn_bwd_stats(const __grid_constant__ BwdParams p) {
  // the main kernel may set itself up meanwhile; it waits for this grid's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.counter = 0u;
  const int bk = blockIdx.x / p.n_sub, st = blockIdx.x - bk * p.n_sub;
  const int b = fast_div(bk, p.by_hkv), kvh = bk - b * p.Hkv;
  const int row = threadIdx.x >> 2, v = threadIdx.x & 3;
  const SubRow r = sub_row(p, st, row);
  const int h = kvh * p.G + r.g;
  float nl = -INFINITY, d = 0.f;
  if (r.valid) {
    const long long at = (static_cast<long long>(b) * p.M + r.m) * p.H + h;
    const float lse = p.lse[at];
    const uint4* x = reinterpret_cast<const uint4*>(p.o + b * p.o_s[0] + r.m * p.o_s[1] + h * p.o_s[2]);
    const uint4* y = reinterpret_cast<const uint4*>(p.d_o + b * p.do_s[0] + r.m * p.do_s[1] + h * p.do_s[2]);
    const uint4 xv[2] = {x[v], x[v + 4]}, yv[2] = {y[v], y[v + 4]};
    uint2 low[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    if (p.o_low != nullptr) {
      const uint2* l = reinterpret_cast<const uint2*>(p.o_low + at * 64);
      low[0] = l[v];
      low[1] = l[v + 4];
    }
    if (lse != -INFINITY) {
      nl = -lse;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float fx[8], fy[8];
        Elem<__nv_bfloat16>::unpack(xv[k], fx);
        Elem<__nv_bfloat16>::unpack(yv[k], fy);
        with_low_bytes(fx, low[k].x);
        with_low_bytes(fx + 4, low[k].y);
#pragma unroll
        for (int i = 0; i < 8; ++i) d += fx[i] * fy[i];
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) d += __shfl_xor_sync(kFullMask, d, o);
  if (v == 0) {
    float* stat = p.stats + static_cast<long long>(blockIdx.x) * kStatFloats;
    stat[row] = nl;
    stat[kSub + row] = -d;
  }
}

struct Barriers {
  uint64_t a_full[kTiles], a_empty[kTiles];  // stationary tiles of an item
  uint64_t b_full[kRing], b_empty[kRing];  // streamed pairs
  uint64_t s_full[kStages], x_full[kStages], t_empty[kStages];
  uint64_t out_full, staged[kTiles], acc_empty, drain[2];
  uint64_t it_full[kQueue], it_empty[kQueue];
  Item item[kQueue];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int kBarrierBytes = 1024;
static_assert(sizeof(Barriers) <= kBarrierBytes, "barrier block");
constexpr int kSmem = kTiles * 4 * kSubBytes + kRing * (2 * kSubBytes + kStatBytes) + kTiles * 2 * kStatBytes +
                      kBarrierBytes + 1024;
static_assert(kSmem <= 227 * 1024, "shared memory");

template <int kMode>
__device__ __forceinline__ Item decode_item(const BwdParams& p, int id) {
  Item it{};
  it.dkv = id < p.n_dkv;
  const int at = it.dkv ? id : id - p.n_dkv, parts = it.dkv ? p.kv_parts : p.q_parts;
  const int i = fast_div(at, it.dkv ? p.by_kv_parts : p.by_q_parts);
  // blk: key block, or pair of sub-tiles counted from the last, whose rows see
  // the most keys under a staircase, as the first keys are seen by the most rows
  const FastDiv& inner = it.dkv ? p.by_kblk : p.by_pair;
  const int outer = fast_div(i, p.bk_inner ? p.by_bk : inner);
  const int rest = i - outer * (p.bk_inner ? p.n_bk : static_cast<int>(inner.d));
  const int blk = p.bk_inner ? outer : rest, bk = p.bk_inner ? rest : outer;
  it.b = fast_div(bk, p.by_hkv);
  it.kvh = bk - it.b * p.Hkv;
  it.L = kMode == kMaskLength ? length_of(p, it.b) : 0;
  if (it.dkv) {
    // position blocks [mt_lo, mt_hi) holding a row that sees a key of the item
    it.k0 = blk * kKeys;
    int mt_lo = 0, mt_hi = p.n_mt;
    if (kMode == kMaskLength) {
      mt_hi = it.k0 < it.L ? min(p.n_mt, static_cast<int>(fast_div(it.L + p.MT - 1, p.by_mt))) : 0;
    } else if (kMode == kMaskAnalytic) {
      const int pe = min(it.k0 + kKeys, p.P);  // prefix keys of the item: [k0, pe)
      const bool prefix = it.k0 < min(pe, p.ds) || max(it.k0, p.de) < pe;
      if (!prefix) {
        const int c = max(it.k0, p.P);  // the first staircase key: visible from row c - (N - M)
        mt_lo = c < min(it.k0 + kKeys, p.N)
                    ? min(p.n_mt, static_cast<int>(fast_div(max(0, c - (p.N - p.M)), p.by_mt)))
                    : p.n_mt;
      }
    }
    it.mt_lo = mt_lo;
    it.mt_hi = mt_hi;
    it.live = p.n_hblk * max(0, mt_hi - mt_lo);
  } else {
    row_item<kMode>(p, blk, it);
  }
  if (parts > 1) take_part(it, at - i * parts, parts);
  return it;
}

// (every warp of the warpgroups behind the compute warps)
__device__ __forceinline__ void less_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
}

template <int kMode, bool kFine>
__global__ void __launch_bounds__(kThreads, 1) attn_bwd(const __grid_constant__ BwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* a_smem = smem;                             // [kTiles][A0 16 KB, A1 16 KB]; then the staged output
  uint8_t* b_smem = a_smem + kTiles * 4 * kSubBytes;       // [kRing][B0 8 KB, B1 8 KB]
  float* b_stat = reinterpret_cast<float*>(b_smem + kRing * 2 * kSubBytes);  // [kRing][128]: dkv
  float* a_stat = b_stat + kRing * kStatFloats;       // [kTiles][2 sub-tiles][128]: dq
  Barriers* bars = reinterpret_cast<Barriers*>(a_stat + kTiles * 2 * kStatFloats);
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
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(&bars->it_full[i], 1);
      mbar_init(&bars->it_empty[i], kComputeWarps + 3 + kOutputWarps);
    }
    mbar_init(&bars->out_full, 1);
    mbar_init(&bars->acc_empty, kOutputWarps);
    mbar_init(&bars->drain[0], 1);
    mbar_init(&bars->drain[1], 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpAccum) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  // Rows of the ring that no query box covers meet P = dS = 0 in the dkv
  // products; clear them once, so that they are finite. (dq steps, which fill
  // whole tiles, only follow the dkv items.)
  {
    const int row0 = p.Gb * p.MT, n = (kSub - row0) * 8;
    for (int i = threadIdx.x; i < 2 * kRing * n; i += kThreads) {
      const int t = i / n;
      reinterpret_cast<uint4*>(b_smem + t * kSubBytes + row0 * kRowBytes)[i - t * n] =
          make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // an allocation of all 512 columns starts at the first; as a constant, it keeps
  // the issue warps' operands uniform
  constexpr uint32_t tmem = 0;

  // The n-th item handed out (live < 0: no more); every warp but the producer
  // takes each once.
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
    // the statistics and the counter are those of the kernel before
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t t = 0, live = 0;  // steps and live items issued
    unsigned next = lane == 0 ? atomicAdd(p.counter, 1u) : 0u;  // taken one ahead: it is a round trip
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t q = n % kQueue;
      if (!__all_sync(kFullMask, bounded_wait(&bars->it_empty[q], ((n / kQueue) & 1) ^ 1, abort_flag)))
        break;
      const int id = min(__shfl_sync(kFullMask, next, 0), static_cast<unsigned>(p.n_items));
      if (lane == 0 && id < p.n_items) next = atomicAdd(p.counter, 1u);
      Item it{};
      if (id < p.n_items)
        it = decode_item<kMode>(p, id);
      else
        it.live = -1;
      if (lane == 0) {
        bars->item[q] = it;
        mbar_arrive(&bars->it_full[q]);
      }
      __syncwarp();
      if (it.live < 0) break;
      if (it.live == 0) continue;
      const int bk = it.b * p.Hkv + it.kvh;
      const uint32_t ab = live % kTiles;
      if (!__all_sync(kFullMask, bounded_wait(&bars->a_empty[ab], ((live / kTiles) & 1) ^ 1, abort_flag)))
        break;
      uint8_t* a0 = a_smem + ab * 4 * kSubBytes;
      uint8_t* a1 = a0 + 2 * kSubBytes;
      if (it.dkv) {
        mbar_arrive_expect_tx_elect(&bars->a_full[ab], 4 * kSubBytes);
        tma_load_4d_elect(a0, &p.tm_k, &bars->a_full[ab], 0, it.kvh, it.k0, it.b);
        tma_load_4d_elect(a1, &p.tm_v, &bars->a_full[ab], 0, it.kvh, it.k0, it.b);
      } else {
        mbar_arrive_expect_tx_elect(
            &bars->a_full[ab],
            static_cast<uint32_t>(it.n_here * (2 * p.Gb * p.MT * kRowBytes + kStatBytes)));
        for (int i = 0; i < it.n_here; ++i) {
          const int hb = fast_div(it.s0 + i, p.by_mt_count), m0 = (it.s0 + i - hb * p.n_mt) * p.MT;
          const int h = it.kvh * p.G + hb * p.Gb;
          tma_load_4d_elect(a0 + i * kSubBytes, &p.tm_q, &bars->a_full[ab], 0, h, m0, it.b);
          tma_load_4d_elect(a1 + i * kSubBytes, &p.tm_do, &bars->a_full[ab], 0, h, m0, it.b);
        }
        bulk_load(a_stat + ab * 2 * kStatFloats,
                  p.stats + (static_cast<long long>(bk) * p.n_sub + it.s0) * kStatFloats,
                  it.n_here * kStatBytes, &bars->a_full[ab]);
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
        uint8_t* b1 = b0 + kSubBytes;
        if (it.dkv) {
          const int m0 = step.pos * p.MT, h = it.kvh * p.G + step.hb * p.Gb;
          mbar_arrive_expect_tx_elect(&bars->b_full[s],
                                      static_cast<uint32_t>(2 * p.Gb * p.MT * kRowBytes + kStatBytes));
          tma_load_4d_elect(b0, &p.tm_q, &bars->b_full[s], 0, h, m0, it.b);
          tma_load_4d_elect(b1, &p.tm_do, &bars->b_full[s], 0, h, m0, it.b);
          bulk_load(b_stat + s * kStatFloats,
                    p.stats + (static_cast<long long>(bk) * p.n_sub + step.hb * p.n_mt + step.pos) * kStatFloats,
                    kStatBytes, &bars->b_full[s]);
        } else {
          mbar_arrive_expect_tx_elect(&bars->b_full[s], 2 * kSubBytes);
          tma_load_4d_elect(b0, &p.tm_k64, &bars->b_full[s], 0, it.kvh, step.pos * kChunk, it.b);
          tma_load_4d_elect(b1, &p.tm_v64, &bars->b_full[s], 0, it.kvh, step.pos * kChunk, it.b);
        }
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
    // T0 = A0 B0^T and T1 = A1 B1^T of every step, up to kStages steps (and one
    // item, by the stationary tiles) ahead of the accumulating products.
    const uint32_t id_kk = idesc_bf16_f32(128, 64, false);
    const uint64_t a_desc = sdesc_sw128(smem_u32(a_smem)), b_desc = sdesc_sw128(smem_u32(b_smem));
    // streamed rows that meet X = 0 only, and may hold NaN, are cleared: keys
    // that no query sees (dq), query rows past L or that see no key (dkv): under a
    // staircase behind nothing but dead keys the first `unseeing` positions
    const int unseeing = kMode == kMaskAnalytic && p.ds == 0 && p.de == p.P ? max(0, p.P - (p.N - p.M)) : 0;
    const bool dead = kMode == kMaskLength || (kMode == kMaskAnalytic && (p.ds < p.de || unseeing > 0));
    Turn<kTiles> ab;
    Turn<kRing> s;
    Turn<kStages> st;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->a_full[ab.i], ab.round, abort_flag))) break;
      const uint64_t a0 = a_desc + ab.i * (4 * kSubBytes / 16), a1 = a0 + 2 * kSubBytes / 16;
      ab.next();
      Steps step;
      step.begin(it);
      for (int j = 0; j < it.live; ++j) {
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->t_empty[st.i], st.round ^ 1, abort_flag) &&
                                       bounded_wait<1>(&bars->b_full[s.i], s.round, abort_flag))) {
          ok = false;
          break;
        }
        if (dead) {
          uint8_t* bp = b_smem + s.i * 2 * kSubBytes;
          if (!it.dkv) {
            const int c0 = step.pos * kChunk;
            const int lo = kMode == kMaskLength ? it.L - c0 : p.ds - c0;
            const int hi = kMode == kMaskLength ? kChunk : p.de - c0;
            clear_rows(bp, max(lo, 0), min(hi, kChunk));
          } else {
            // rows of the step's positions before L, or before the first that sees
            const int n = (kMode == kMaskLength ? it.L : unseeing) - step.pos * p.MT;
            const int before = min(min(max(n, 0), kSub) * p.Gb, kSub);
            const int lo = kMode == kMaskLength ? before : 0, hi = kMode == kMaskLength ? kSub : before;
            clear_rows(bp, lo, hi);
            clear_rows(bp + kSubBytes, lo, hi);
          }
          step.next(it);
        }
        tc_fence_after();
        const uint64_t b0 = b_desc + s.i * (2 * kSubBytes / 16);
        const uint32_t d = tmem + kStage0 + st.i * kStageCols;
        umma_ss_x4(d, a0, b0, id_kk);
        umma_ss_x4(d + kT1, a1, b0 + kSubBytes / 16, id_kk);
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
    // acc1 += X1 B0, and acc0 += X0 B1 of a dkv item.
    const uint32_t id_kn = idesc_bf16_f32(128, 64, true);
    const uint64_t b_desc = sdesc_sw128(smem_u32(b_smem));
    Turn<kRing> s;
    Turn<kStages> st;
    uint32_t live = 0;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      // the previous item's accumulators have been read
      if (live > 0 &&
          !__all_sync(kFullMask, bounded_wait<1>(&bars->acc_empty, (live - 1) & 1, abort_flag)))
        break;
      for (int j = 0; j < it.live; ++j) {
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->x_full[st.i], st.round, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t b0 = b_desc + s.i * (2 * kSubBytes / 16);
        const uint32_t x = tmem + kStage0 + st.i * kStageCols;
        umma_ts_x4(tmem + kAcc0, x, b0 + kSubBytes / 16, id_kn, j > 0, it.dkv);  // dV += P^T dO
        umma_ts_x4(tmem + kAcc1, x + kT1, b0, id_kn, j > 0, 1u);  // dK += dS^T Q, dQ += dS K
        if (kFine) {  // the rests of P and dS
          umma_ts_x4(tmem + kAcc0, x + 8, b0 + kSubBytes / 16, id_kn, 1u, it.dkv);
          umma_ts_x4(tmem + kAcc1, x + kT1 + 8, b0, id_kn, 1u, 1u);
        }
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsCompute));
    // Compute warps. A step belongs to the group of its parity.
    const int group = warp >> 3, quarter = warp & 3, gq = (warp >> 2) & 1;
    const int tl = quarter * 32 + lane;  // TMEM lane: key of a dkv item, row of a dq item
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
    uint32_t t = 0, live = 0;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      // this lane's key, or row
      const int key = it.k0 + tl;
      const SubRow r = sub_row(p, it.s0 + (quarter >> 1), (quarter & 1) * 32 + lane);
      const bool valid = it.dkv ? key < p.N : r.valid;
      const uint32_t ab = live % kTiles;
      // dkv: rows m in [from, to) see the key; dq: keys [0, from) and [mid, to)
      // are seen by the row
      int from = 0, mid = 0, to = 0;
      if (it.dkv) {
        to = p.M;
        if (kMode == kMaskAnalytic) {
          if (key >= p.P)
            from = key - (p.N - p.M);
          else if (key >= p.ds && key < p.de)
            to = 0;
        } else if (kMode == kMaskLength) {
          to = key < it.L ? it.L : 0;
        }
        if (!valid) to = 0;
      } else {
        if (kMode == kMaskAnalytic) {
          from = p.ds;
          mid = p.de;
          to = max(p.P, min(p.N, p.N - p.M + r.m + 1));
        } else if (kMode == kMaskLength) {
          to = r.m < it.L ? it.L : 0;
        }
      }
      // A step's 32 columns of this warp, by their first key c (dq) or the
      // sub-tile's first position c (dkv), are seen by all its lanes when
      // c <= all_0 or all_1 <= c <= all_2, and by none when no_0 <= c <= no_1 or
      // c >= no_2; lanes without a key or row do not count.
      constexpr int kFar = INT32_MAX / 2;
      int all_0 = -kFar, all_1 = 0, all_2 = 0, no_0 = -kFar, no_1 = 0, no_2 = 0;
      if (kMode != kMaskBool) {
        const int to_lo = __reduce_min_sync(kFullMask, valid ? to : kFar);
        const int to_hi = __reduce_max_sync(kFullMask, valid ? to : -kFar);
        if (it.dkv) {
          // column of position m: (m - c) Gb - 32 gq
          const int before = 32 * gq / p.Gb, past = (32 * gq + 32 + p.Gb - 1) / p.Gb;
          all_1 = __reduce_max_sync(kFullMask, valid ? from : -kFar) - before;
          all_2 = to_lo >= p.M ? kFar : to_lo - past;
          no_1 = __reduce_min_sync(kFullMask, valid ? from : kFar) - past;
          no_2 = to_hi - before;
        } else {
          all_0 = from - 32;
          all_1 = mid;
          all_2 = to_lo - 32;
          no_0 = from;
          no_1 = mid - 32;
          no_2 = max(from, to_hi);
        }
      }
      uint64_t nl2 = 0ull, nD2 = 0ull;
      // this group's steps: every other one
      const int j0 = static_cast<int>((t ^ group) & 1u);
      if (!it.dkv && j0 < it.live) {
        // the row's statistics (only with a step to do: a group without one may
        // come here after the tiles have been replaced)
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->a_full[ab], (live / kTiles) & 1, abort_flag))) break;
        const float* stat = a_stat + (ab * 2 + (quarter >> 1)) * kStatFloats + (quarter & 1) * 32 + lane;
        nl2 = f2_pack(stat[0], stat[0]);
        nD2 = f2_pack(stat[kSub], stat[kSub]);
      }
      const int per_head = it.mt_hi - it.mt_lo;  // position blocks of a head block (dkv)
      int pos = it.mt_lo + j0 + (it.dkv && it.j0 > 0 ? it.j0 % per_head : 0);
      for (int j = j0; j < it.live; j += 2, pos += 2) {
        int c;
        if (it.dkv) {
          while (pos >= it.mt_hi) pos -= per_head;
          c = pos * p.MT;
        } else {
          const int k = it.j0 + j;
          c = (k < it.a1 ? k : k - it.a1 + it.b0) * kChunk + 32 * gq;
        }
        // which of the columns this lane sees (dkv: rows past M or the box have
        // -lse = -inf, so their P is 0 without a mask)
        uint32_t vm = 0u;
        bool full, none;
        if (kMode == kMaskBool) {
          if (it.dkv && valid) {
            // the positions of the warp's columns, each spread over Gb of them
            // (the first may have begun in the columns before)
            const int first = 32 * gq / p.Gb, begun = 32 * gq - first * p.Gb;
            if (first < p.MT && c + first < p.M) {
              const uint32_t seen = col_bits_at(p, it.b, key, c + first);
              if (p.Gb == 1) {
                vm = seen;
              } else {
                const uint64_t heads = ~0ull >> (64 - p.Gb);
                const int last = min(p.MT - first, (32 + begun + p.Gb - 1) / p.Gb);
                for (int i = 0; i < last; ++i)
                  if ((seen >> i) & 1u) vm |= static_cast<uint32_t>((heads << (i * p.Gb)) >> begun);
              }
            }
          } else if (!it.dkv && valid && c < p.N) {
            vm = row_bits_at(p, it.b, r.m, c);
          }
          full = __all_sync(kFullMask, !valid || vm == 0xffffffffu);
          none = __all_sync(kFullMask, !valid || vm == 0u);
        } else {
          full = c <= all_0 || (c >= all_1 && c <= all_2);
          none = (c >= no_0 && c <= no_1) || c >= no_2;
          if (!full && !none) {
            if (it.dkv) {
              auto column = [&](int m) { return min(max(m - c, 0), kSub) * p.Gb - 32 * gq; };
              vm = ~low_bits(column(from)) & (to >= p.M ? 0xffffffffu : low_bits(column(to)));
            } else {
              vm = low_bits(from - c) | (low_bits(to - c) & ~low_bits(mid - c));
            }
          }
        }
        const uint32_t tj = t + j, st = tj % kStages, s = tj % kRing;
        // A group sees every phase of its ring slots (kRing is even), and a
        // stage's skipped phase completes before the step it sees in between.
        if (!__all_sync(kFullMask,
                        (!it.dkv || bounded_wait<1>(&bars->b_full[s], (tj / kRing) & 1, abort_flag)) &&
                            bounded_wait<1>(&bars->s_full[st], (tj / kStages) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t0 = tbase + kStage0 + st * kStageCols + 32 * gq;
        if (none) {
          const uint32_t zero[8] = {};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (it.dkv) tmem_st8(t0 + 16 * h, zero);
            tmem_st8(t0 + kT1 + 16 * h, zero);
            if (kFine) {
              if (it.dkv) tmem_st8(t0 + 16 * h + 8, zero);
              tmem_st8(t0 + kT1 + 16 * h + 8, zero);
            }
          }
        } else {
          const float4* stat = reinterpret_cast<const float4*>(b_stat + s * kStatFloats) + 8 * gq;
          // Sixteen columns at a time, which keeps the step in registers. Four
          // bodies: per-column or per-lane statistics, all shown or not.
          auto grads = [&](auto dkv, auto masked) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float sv[16], dp[16];
              tmem_ld16(t0 + 16 * h, sv);
              tmem_ld16(t0 + kT1 + 16 * h, dp);
              tmem_wait_ld();
              uint32_t pp[8], pd[8], rp[4], rd[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {  // four columns
                uint64_t l2[2] = {nl2, nl2}, d2[2] = {nD2, nD2};
                if (decltype(dkv)::value) {
                  const float4 l4 = stat[4 * h + i], d4 = stat[16 + 4 * h + i];
                  l2[0] = f2_pack(l4.x, l4.y);
                  l2[1] = f2_pack(l4.z, l4.w);
                  d2[0] = f2_pack(d4.x, d4.y);
                  d2[1] = f2_pack(d4.z, d4.w);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  const int k = 2 * i + u;
                  float x0, x1, d0, d1;
                  f2_unpack(f2_fma(f2_pack(sv[2 * k], sv[2 * k + 1]), sl2, l2[u]), x0, x1);
                  float e0 = ex2(x0), e1 = ex2(x1);
                  f2_unpack(f2_mul(f2_pack(e0, e1),
                                   f2_add(f2_pack(dp[2 * k], dp[2 * k + 1]), d2[u])), d0, d1);
                  if (decltype(masked)::value) {
                    const uint32_t bits = vm >> (16 * h + 2 * k);
                    e0 = bits & 1u ? e0 : 0.f;
                    d0 = bits & 1u ? d0 : 0.f;
                    e1 = bits & 2u ? e1 : 0.f;
                    d1 = bits & 2u ? d1 : 0.f;
                  }
                  if (decltype(dkv)::value) pp[k] = pack_bf16x2(e0, e1);
                  pd[k] = pack_bf16x2(d0, d1);
                  if (kFine) {
                    if (decltype(dkv)::value) rp[k % 4] = rest_of_pair(e0, e1, pp[k]);
                    rd[k % 4] = rest_of_pair(d0, d1, pd[k]);
                  }
                }
                if (kFine && i % 2 == 1) {
                  // over the columns just read, the rests behind
                  const uint32_t at = t0 + 16 * h + 4 * (i / 2);
                  if (decltype(dkv)::value) tmem_st4(at, pp + 2 * i - 2);
                  if (decltype(dkv)::value) tmem_st4(at + 8, rp);
                  tmem_st4(at + kT1, pd + 2 * i - 2);
                  tmem_st4(at + kT1 + 8, rd);
                }
              }
              if (!kFine) {
                if (decltype(dkv)::value) tmem_st8(t0 + 16 * h, pp);
                tmem_st8(t0 + kT1 + 16 * h, pd);
              }
            }
          };
          using Yes = std::true_type;
          using No = std::false_type;
          if (it.dkv)
            full ? grads(Yes(), No()) : grads(Yes(), Yes());
          else
            full ? grads(No(), No()) : grads(No(), Yes());
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_elect(&bars->x_full[st]);
      }
      t += it.live;
      ++live;
    }
  } else if (warp >= kWarpOutput) {
    less_registers();
    // Outputs: the accumulators, scaled, staged over the item's stationary tiles
    // in the swizzled layout of the maps. One lane quarter of
    // TMEM per warp.
    const int quarter = warp & 3;
    const int tl = quarter * 32 + lane;  // key of a dkv item, row of a dq item
    const uint32_t tbase = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    uint32_t live = 0;
    Turn<kTiles> ab;
    for (uint32_t n = 0;; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      const int parts = it.dkv ? p.kv_parts : p.q_parts;
      // this lane's sums of a part: 128 (dK, dV) or 64 (dQ) of them
      float* sums = nullptr;
      if (parts > 1) {
        const int bk = it.b * p.Hkv + it.kvh;
        if (it.dkv)
          sums = p.kv_sums + ((static_cast<long long>(it.part) * p.n_bk + bk) * p.n_kblk * kKeys +
                              it.k0 + tl) * 128;
        else if ((quarter >> 1) < it.n_here)
          sums = p.q_sums + ((static_cast<long long>(it.part) * p.n_bk + bk) * p.n_sub * kSub +
                             static_cast<long long>(it.s0) * kSub + tl) * 64;
      }
      if (it.live == 0) {  // nothing seen: zeros
        const int key = it.k0 + tl;
        const SubRow r = sub_row(p, it.s0 + (quarter >> 1), (quarter & 1) * 32 + lane);
        if (sums != nullptr) {
          for (int v = 0; v < (it.dkv ? 32 : 16); ++v)
            reinterpret_cast<float4*>(sums)[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (parts == 1 && (it.dkv ? key < p.N : r.valid)) {
          const long long at =
              it.dkv ? ((static_cast<long long>(it.b) * p.N + key) * p.Hkv + it.kvh) * 64
                     : ((static_cast<long long>(it.b) * p.M + r.m) * p.H + it.kvh * p.G + r.g) * 64;
          uint4* d0 = reinterpret_cast<uint4*>((it.dkv ? p.dk : p.dq) + at);
          uint4* d1 = reinterpret_cast<uint4*>((it.dkv ? p.dv : p.dq) + at);
#pragma unroll
          for (int v = 0; v < 8; ++v) d0[v] = d1[v] = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->out_full, live & 1, abort_flag))) break;
      tc_fence_after();
      uint8_t* a0 = a_smem + ab.i * 4 * kSubBytes;
      // dK over K (dQ over Q), then dV over V, 32 columns at a time
      const int blocks = it.dkv ? 4 : 2;
#pragma unroll 1
      for (int q = 0; q < blocks; ++q) {
        const bool dv = q >= 2;
        float o[2][16];
        tmem_ld16(tbase + (dv ? kAcc0 - 64 : kAcc1) + 32 * q, o[0]);
        tmem_ld16(tbase + (dv ? kAcc0 - 64 : kAcc1) + 32 * q + 16, o[1]);
        tmem_wait_ld();
        if (q == blocks - 1) {  // read: the next item may accumulate
          tc_fence_before();
          mbar_arrive_elect(&bars->acc_empty);
        }
        if (parts > 1) {
          if (sums != nullptr) {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              reinterpret_cast<float4*>(sums)[8 * q + v] =
                  make_float4(o[v / 4][v % 4 * 4], o[v / 4][v % 4 * 4 + 1], o[v / 4][v % 4 * 4 + 2],
                              o[v / 4][v % 4 * 4 + 3]);
          }
        } else {
          const float scale = dv ? 1.f : scale_of(p, it.L);
          uint8_t* stage = a0 + (dv ? 2 * kSubBytes : 0) + tl * kRowBytes;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_bf16x2(o[v / 2][v % 2 * 8 + 2 * e] * scale, o[v / 2][v % 2 * 8 + 2 * e + 1] * scale);
            const uint32_t c = static_cast<uint32_t>(4 * (q & 1) + v) ^ static_cast<uint32_t>(tl & 7);
            st_shared_v4(stage + c * 16, w[0], w[1], w[2], w[3]);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(&bars->staged[ab.i]);
      ab.next();
      ++live;
    }
  } else {
    less_registers();
    // Stores of the staged outputs, which release the items' tiles. A tile's
    // barrier is not arrived at again before the tile has been released.
    Turn<kTiles> ab;
    for (uint32_t n = 0;; ++n) {
      Item it;
      if (!take_item(n, it) || it.live < 0) break;
      if (it.live == 0) continue;
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->staged[ab.i], ab.round, abort_flag))) break;
      if (lane == 0) {
        if ((it.dkv ? p.kv_parts : p.q_parts) == 1) {
          uint8_t* a0 = a_smem + ab.i * 4 * kSubBytes;
          if (it.dkv) {
            tma_store_4d(&p.tm_dk, a0, 0, it.kvh, it.k0, it.b);
            tma_store_4d(&p.tm_dv, a0 + 2 * kSubBytes, 0, it.kvh, it.k0, it.b);
          } else {
            for (int i = 0; i < it.n_here; ++i) {
              const int hb = fast_div(it.s0 + i, p.by_mt_count), m0 = (it.s0 + i - hb * p.n_mt) * p.MT;
              tma_store_4d(&p.tm_dq, a0 + i * kSubBytes, 0, it.kvh * p.G + hb * p.Gb, m0, it.b);
            }
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

// ---------------------------------------------------------------------------
// Joins of parts: the sums of an output, in the order of the parts, scaled and
// rounded; four sums per thread. Bound: HBM, one read of the sums.
__device__ __forceinline__ float4 sum_parts(const float* at, long long part_stride, int parts) {
  float4 s = *reinterpret_cast<const float4*>(at);
#pragma unroll 4
  for (int k = 1; k < parts; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(at + k * part_stride);
    s.x += x.x;
    s.y += x.y;
    s.z += x.z;
    s.w += x.w;
  }
  return s;
}
__device__ __forceinline__ void store_4(__nv_bfloat16* dst, float4 s, float scale) {
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(pack_bf16x2(s.x * scale, s.y * scale), pack_bf16x2(s.z * scale, s.w * scale));
}
// blockIdx.y: (b, kv head); 32 threads per key: dK, then dV
__global__ void __launch_bounds__(256) attn_bwd_join_kv(const __grid_constant__ BwdParams p) {
  const int key = blockIdx.x * 8 + (threadIdx.x >> 5), bk = blockIdx.y, v = threadIdx.x & 31;
  if (key >= p.N) return;
  const long long rows = static_cast<long long>(p.n_kblk) * kKeys;
  const float4 s = sum_parts(p.kv_sums + (bk * rows + key) * 128 + 4 * v, p.n_bk * rows * 128, p.kv_parts);
  const int b = fast_div(bk, p.by_hkv), kvh = bk - b * p.Hkv;
  const long long at = ((static_cast<long long>(b) * p.N + key) * p.Hkv + kvh) * 64 + 4 * (v & 15);
  const int L = p.lengths != nullptr ? length_of(p, b) : 0;
  store_4((v < 16 ? p.dk : p.dv) + at, s, v < 16 ? scale_of(p, L) : 1.f);
}
// blockIdx.y: (b, kv head), blockIdx.x: quarter of a sub-tile; 16 threads per row
__global__ void __launch_bounds__(256) attn_bwd_join_q(const __grid_constant__ BwdParams p) {
  const int st = blockIdx.x >> 2, row = (blockIdx.x & 3) * 16 + (threadIdx.x >> 4);
  const int bk = blockIdx.y, v = threadIdx.x & 15;
  const SubRow r = sub_row(p, st, row);
  if (!r.valid) return;
  const long long rows = static_cast<long long>(p.n_sub) * kSub;
  const float4 s = sum_parts(p.q_sums + (bk * rows + static_cast<long long>(st) * kSub + row) * 64 + 4 * v,
                             p.n_bk * rows * 64, p.q_parts);
  const int b = fast_div(bk, p.by_hkv), kvh = bk - b * p.Hkv;
  const int L = p.lengths != nullptr ? length_of(p, b) : 0;
  store_4(p.dq + ((static_cast<long long>(b) * p.M + r.m) * p.H + kvh * p.G + r.g) * 64 + 4 * v, s,
          scale_of(p, L));
}

// ---------------------------------------------------------------------------
// host

// Parts and workspace of a call: the sub-tiles' statistics, the item counter, the
// parts' sums, and the packed mask.
struct BwdPlan {
  SubTiling tl;
  int64_t n_bk, n_kblk, n_pair;
  int kv_parts, q_parts;
  bool fine;
  int64_t counter, kv_sums, q_sums, row_bits, col_bits, bytes;  // offsets and size
};
BwdPlan plan_bwd(const vlak_attn_gqa_args* a, bool keys_too, bool masked) {
  BwdPlan w{};
  w.tl = sub_tiling(static_cast<int>(a->H / a->Hkv), static_cast<int>(a->M));
  w.n_bk = a->B * a->Hkv;
  w.n_kblk = (a->N + kKeys - 1) / kKeys;
  w.n_pair = (w.tl.n_sub + 1) / 2;
  const int64_t n_chunks = (a->N + kChunk - 1) / kChunk;
  const int64_t total = w.n_bk * (w.n_pair * n_chunks + (keys_too ? w.n_kblk * w.tl.n_sub : 0));
  w.kv_parts = keys_too ? item_parts(w.tl.n_sub, total) : 1;
  w.q_parts = item_parts(n_chunks, total);
  w.fine = fine_call(*a, total);
  w.counter = w.n_bk * w.tl.n_sub * kStatBytes;
  w.kv_sums = w.counter + 256;
  w.q_sums = w.kv_sums + (w.kv_parts > 1 ? w.kv_parts * w.n_bk * w.n_kblk * kKeys * 128 * 4 : 0);
  w.row_bits = w.q_sums + (w.q_parts > 1 ? w.q_parts * w.n_bk * w.tl.n_sub * kSub * 64 * 4 : 0);
  w.col_bits = w.row_bits + (masked ? row_bits_bytes(*a) : 0);
  w.bytes = w.col_bits + (masked && keys_too ? col_bits_bytes(*a) : 0);
  return w;
}

template <int kMode, bool kFine>
cudaError_t launch_both(const BwdParams& p, unsigned n_stats, unsigned grid, cudaStream_t cs, int device) {
  static std::atomic<int> ready[64];
  if (ready[device].load() == 0) {
    cudaError_t e = cudaFuncSetAttribute(attn_bwd<kMode, kFine>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kSmem);
    if (e != cudaSuccess) return e;
    ready[device].store(1);
  }
  attn_bwd_stats<<<n_stats, kStatThreads, 0, cs>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // programmatic dependent launch: set up while the statistics are computed
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = cs;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, attn_bwd<kMode, kFine>, p);
  if (e == cudaSuccess && p.kv_parts > 1) {
    attn_bwd_join_kv<<<dim3((p.N + 7) / 8, p.n_bk), 256, 0, cs>>>(p);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess && p.q_parts > 1) {
    attn_bwd_join_q<<<dim3(p.n_sub * 4, p.n_bk), 256, 0, cs>>>(p);
    e = cudaGetLastError();
  }
  return e;
}

int bwd_validate(const vlak_attn_train_args* a, int64_t* P, float* scale) {
  if (!a) return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: null arguments");
  int st = check_train(&a->attn, P, scale, "fused_attention_gqa_bwd");
  if (st != VLAK_OK) return st;
  const void* ptrs[4] = {a->grad_o, a->dq, a->dk, a->dv};
  for (const void* ptr : ptrs)
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: pointers must be 16-byte aligned");
  for (int d = 0; d < 3; ++d)
    if (a->grad_o_stride[d] % 8 != 0)
      return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: grad_o strides must be multiples of 8");
  if (reinterpret_cast<uintptr_t>(a->lse) % 4 != 0 || reinterpret_cast<uintptr_t>(a->o_low) % 16 != 0)
    return set_error(VLAK_ERR_ALIGNMENT,
                     "fused_attention_gqa_bwd: lse must be 4-byte, o_low 16-byte aligned");
  return check_train_masks(*a, "fused_attention_gqa_bwd");
}

int run_bwd(const vlak_attn_train_args* t, void* workspace, int64_t ws_bytes, void* stream) {
  clear_error();
  vlak_attn_train_args args{};
  if (t) {
    args = *t;
    if (args.lengths || args.mask) {
      args.attn.prefix_len = -1;
      args.attn.dead_start = args.attn.dead_end = 0;
    }
  }
  int64_t P = 0;
  float scale = 0.f;
  int st = bwd_validate(t ? &args : nullptr, &P, &scale);
  if (st != VLAK_OK) return st;
  const vlak_attn_gqa_args* a = &args.attn;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int64_t q_rows = a->B * a->M * a->H, k_rows = a->B * a->N * a->Hkv;
  const bool keys_too = args.dk || args.dv;  // else dq alone
  if ((q_rows > 0 && !args.dq) || (k_rows > 0 && keys_too && (!args.dk || !args.dv)))
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: null gradient pointer");
  if (q_rows == 0 || k_rows == 0) {  // nothing sees anything
    cudaError_t e = cudaSuccess;
    if (q_rows > 0) e = cudaMemsetAsync(args.dq, 0, q_rows * 128, cs);
    if (k_rows > 0 && keys_too && e == cudaSuccess) e = cudaMemsetAsync(args.dk, 0, k_rows * 128, cs);
    if (k_rows > 0 && keys_too && e == cudaSuccess) e = cudaMemsetAsync(args.dv, 0, k_rows * 128, cs);
    return e == cudaSuccess ? VLAK_OK : set_cuda_error("fused_attention_gqa_bwd zero fill", e);
  }
  if (!a->q || !a->k || !a->v || !a->o || !args.grad_o || !args.lse)
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: null tensor pointer");
  const BwdPlan plan = plan_bwd(a, keys_too, args.mask != nullptr);
  if (!workspace || ws_bytes < plan.bytes)
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: workspace missing or too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: workspace must be 256-byte aligned");
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != VLAK_OK) return st;
  if (dev.cc_major != 10)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DEVICE,
                      "fused_attention_gqa_bwd: needs an sm_100 device (found sm_%d%d)", dev.cc_major,
                      dev.cc_minor);
  if (dev.device >= 64) return set_error(VLAK_ERR_CUDA, "device ordinal out of range");

  BwdParams p;
  memset(&p, 0, sizeof(p));
  const SubTiling& tl = plan.tl;
  const int64_t n_bk = plan.n_bk, n_dq = n_bk * plan.n_pair * plan.q_parts;
  const int64_t n_dkv = keys_too ? n_bk * plan.n_kblk * plan.kv_parts : 0;
  if (n_dq + n_dkv > INT32_MAX - 4096 || n_bk * tl.n_sub > INT32_MAX)
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: too many work items");
  static_cast<TrainShape&>(p) = train_shape(a, P, scale, tl);
  set_masks(p, args);
  p.n_kblk = static_cast<int>(plan.n_kblk);
  p.n_dkv = static_cast<int>(n_dkv);
  p.n_items = static_cast<int>(n_dkv + n_dq);
  p.kv_parts = plan.kv_parts;
  p.q_parts = plan.q_parts;
  p.by_kblk = fast_div_by(static_cast<unsigned>(p.n_kblk));
  p.by_kv_parts = fast_div_by(static_cast<unsigned>(p.kv_parts));
  p.by_q_parts = fast_div_by(static_cast<unsigned>(p.q_parts));
  // the last row sees the most keys: all but the dead ones
  p.out_scale = p.ds + p.N - p.de <= 1 ? 0.f : p.scale;
  p.host_err = host_error_word(cs);
  p.lse = args.lse;
  p.stats = static_cast<float*>(workspace);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counter = reinterpret_cast<unsigned*>(ws + plan.counter);
  p.kv_sums = reinterpret_cast<float*>(ws + plan.kv_sums);
  p.q_sums = reinterpret_cast<float*>(ws + plan.q_sums);
  p.row_bits = reinterpret_cast<uint32_t*>(ws + plan.row_bits);
  p.col_bits = keys_too ? reinterpret_cast<uint32_t*>(ws + plan.col_bits) : nullptr;
  p.o = static_cast<const __nv_bfloat16*>(a->o);
  p.d_o = static_cast<const __nv_bfloat16*>(args.grad_o);
  p.o_low = static_cast<const int8_t*>(args.o_low);
  for (int d = 0; d < 3; ++d) {
    p.o_s[d] = a->o_stride[d];
    p.do_s[d] = args.grad_o_stride[d];
  }
  p.dq = static_cast<__nv_bfloat16*>(args.dq);
  p.dk = static_cast<__nv_bfloat16*>(args.dk);
  p.dv = static_cast<__nv_bfloat16*>(args.dv);
  const uint32_t gb = static_cast<uint32_t>(tl.Gb), mt = static_cast<uint32_t>(tl.MT);
  auto rows = [&](CUtensorMap* m, const void* ptr, const int64_t* s, const char* name) {
    return encode_map(m, ptr, a->H, a->M, a->B, s[2], s[1], s[0], gb, mt, name);
  };
  auto keys = [&](CUtensorMap* m, const void* ptr, const int64_t* s, uint32_t box, const char* name) {
    return encode_map(m, ptr, a->Hkv, a->N, a->B, s[2], s[1], s[0], 1, box, name);
  };
  const int64_t qs[3] = {a->M * a->H * 64, a->H * 64, 64}, ks[3] = {a->N * a->Hkv * 64, a->Hkv * 64, 64};
  st = rows(&p.tm_q, a->q, a->q_stride, "q");
  if (st == VLAK_OK) st = rows(&p.tm_do, args.grad_o, args.grad_o_stride, "grad_o");
  if (st == VLAK_OK) st = rows(&p.tm_dq, args.dq, qs, "dq");
  if (st == VLAK_OK) st = keys(&p.tm_k64, a->k, a->k_stride, kChunk, "k");
  if (st == VLAK_OK) st = keys(&p.tm_v64, a->v, a->v_stride, kChunk, "v");
  if (st != VLAK_OK) return st;
  if (keys_too) st = keys(&p.tm_k, a->k, a->k_stride, kKeys, "k");
  if (keys_too && st == VLAK_OK) st = keys(&p.tm_v, a->v, a->v_stride, kKeys, "v");
  if (keys_too && st == VLAK_OK) st = keys(&p.tm_dk, args.dk, ks, kKeys, "dk");
  if (keys_too && st == VLAK_OK) st = keys(&p.tm_dv, args.dv, ks, kKeys, "dv");
  if (st != VLAK_OK) return st;

  const unsigned n_stats = static_cast<unsigned>(n_bk * p.n_sub);
  const unsigned grid = static_cast<unsigned>(std::min(p.n_items, dev.sm_count));
  cudaError_t e = args.mask ? launch_pack(args, p, cs) : cudaSuccess;
  if (e != cudaSuccess) return set_cuda_error("fused_attention_gqa_bwd mask", e);
  auto launch = [&](auto fine) {
    constexpr bool kFine = decltype(fine)::value;
    return args.lengths ? launch_both<kMaskLength, kFine>(p, n_stats, grid, cs, dev.device)
           : args.mask  ? launch_both<kMaskBool, kFine>(p, n_stats, grid, cs, dev.device)
                        : launch_both<kMaskAnalytic, kFine>(p, n_stats, grid, cs, dev.device);
  };
  e = plan.fine ? launch(std::true_type()) : launch(std::false_type());
  if (e != cudaSuccess) return set_cuda_error("fused_attention_gqa_bwd launch failed", e);
  return VLAK_OK;
}

}  // namespace

int take_bwd_device_error(int* code) { return take_device_error(code); }

}  // namespace vlak

extern "C" int vlak_attn_gqa_bwd_workspace_size(const vlak_attn_train_args* args, int64_t* bytes) {
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
  int st = check_train(&a, nullptr, nullptr, "workspace size");
  if (st != VLAK_OK) return st;
  if (a.B > 0 && a.M > 0 && a.N > 0)
    *bytes = plan_bwd(&a, args->dk || args->dv, args->mask != nullptr).bytes;
  return VLAK_OK;
}

extern "C" int vlak_attn_gqa_bwd(const vlak_attn_train_args* args, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return vlak::run_bwd(args, workspace, workspace_bytes, stream);
}
