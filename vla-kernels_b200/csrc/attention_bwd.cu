// Backward pass of the GQA attention (attention_gqa.cu) for sm_100a: tcgen05
// products with TMEM accumulators, probabilities recomputed from the scores.
//
// Mathematics, per query head with s = q.k (scaled), P = exp(s - logsumexp):
//   dV = P^T dO,  dP = dO V^T,  D = rowsum(dO * O),  dS = P * (dP - D),
//   dQ = scale dS K,  dK = scale dS^T Q,
// dK and dV summed over the G query heads of a kv head. Scores are taken in
// the exp2 domain: P = 2^(scale log2(e) s - lse), lse from the forward pass.
//
// Two kernels, no atomics, so results repeat bit for bit:
//   dq   one CTA per 128 query rows: walks the keys, S = Q K^T, dP = dO V^T,
//        dS in bf16 back to TMEM, dQ += dS K. It also computes D and leaves
//        (-lse, -D) of its rows in the workspace for the second kernel.
//   dkv  one CTA per 128 keys: walks the query rows of all G heads,
//        S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q with
//        P^T and dS^T in TMEM. Keys lie along TMEM lanes, so nothing is ever
//        transposed through shared memory.
// The scores and dP are computed in both (7 products instead of 5): joining
// dQ across key blocks would take atomics or a pass over partial sums.
//
// Rounding: P and dS are rounded to bf16 as operands of the second products,
// as the forward pass rounds P; all sums, D and the statistics are fp32.
//
// Query rows are handled in sub-tiles of up to 64 rows, Gb heads x MT
// positions with Gb a divisor of G, one TMA box each. Two sub-tiles make the
// 128 lanes of a dq CTA; one is the 64 columns of a dkv step.
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

#include "attention_common.cuh"
#include "vlak_device.cuh"
#include "vlak_internal.h"

namespace vlak {
namespace {

constexpr int kMaskAnalytic = 0, kMaskLength = 1, kMaskBool = 2;

constexpr int kSub = 64;                     // query rows of a sub-tile
constexpr int kRowBytes = 128;               // 64 bf16
constexpr int kSubBytes = kSub * kRowBytes;  // 8 KB
constexpr int kChunk = 64;                   // keys of a dq step
constexpr int kKeys = 128;                   // keys of a dkv CTA
constexpr int kDqStages = 3;                 // K/V chunks in flight
constexpr int kDkvStages = 4;                // query sub-tiles in flight
constexpr int kStatBytes = 2 * kSub * 4;     // -lse and -D of a sub-tile
constexpr int kThreads = 192;                // four compute warps, producer, MMA
constexpr int kWarpProducer = 4, kWarpMma = 5;
constexpr uint32_t kTmemCols = 256;
constexpr int kBarrierBytes = 256;

constexpr int kDqSmem = 6 * kSubBytes + kDqStages * 2 * kSubBytes + kBarrierBytes + 1024;
constexpr int kDkvSmem =
    4 * kSubBytes + kDkvStages * (2 * kSubBytes + kStatBytes) + kBarrierBytes + 1024;
static_assert(2 * (kDqSmem + 1024) <= 228 * 1024, "two dq CTAs share an SM");
static_assert(2 * (kDkvSmem + 1024) <= 228 * 1024, "two dkv CTAs share an SM");

struct __align__(64) BwdParams {
  CUtensorMap tm_q, tm_do, tm_o, tm_dq;      // dims (64, H, M, B), box (64, Gb, MT, 1)
  CUtensorMap tm_k64, tm_v64;                // dims (64, Hkv, N, B), box (64, 1, 64, 1)
  CUtensorMap tm_k, tm_v, tm_dk, tm_dv;      // the same, box (64, 1, 128, 1)
  __nv_bfloat16 *dq, *dk, *dv;               // contiguous
  const float* lse;                          // (B, M, H), log2 units
  float* stats;                              // [B * Hkv][n_sub][-lse 64, -D 64]
  int B, M, N, H, Hkv, G;
  int Gb, MT;                                // heads and positions of a sub-tile
  int n_mt, n_sub, n_pair, n_kblk, n_chunks;
  int P, ds, de;
  float scale_log2, out_scale;
  int* host_err;
  const void* lengths;
  int lengths_i64;
  const uint8_t* mask;
  long long mask_sb, mask_sm;
  int mask_words;
};

__device__ __forceinline__ int length_of(const BwdParams& p, int b) {
  const long long len = p.lengths_i64 ? static_cast<const long long*>(p.lengths)[b]
                                      : static_cast<const int*>(p.lengths)[b];
  return static_cast<int>(min(max(len, 0LL), static_cast<long long>(p.N)));
}

// low n bits set, n clamped to [0, 32]
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : ((1u << n) - 1u);
}

// 1024-byte aligned start of the dynamic shared memory
__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) {
  return raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
}

// ---------------------------------------------------------------------------
// dq kernel

struct DqBarriers {
  uint64_t q_full, k_full[kDqStages], k_empty[kDqStages], s_full, ds_full, out_full, staged[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(DqBarriers) <= kBarrierBytes, "barrier block");

// TMEM columns of the dq kernel; dS (bf16 pairs) overwrites the first half of S
constexpr uint32_t kDqS = 0, kDqP = 64, kDqO = 128;

template <int kMode>
__global__ void __launch_bounds__(kThreads, 2) attn_bwd_dq(const __grid_constant__ BwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* q_smem = smem;                      // [2 sub-tiles][64 x 128 B]
  uint8_t* do_smem = q_smem + 2 * kSubBytes;
  uint8_t* o_smem = do_smem + 2 * kSubBytes;   // O, then the staged dQ
  uint8_t* k_smem = o_smem + 2 * kSubBytes;    // [stage][64 x 128 B]
  uint8_t* v_smem = k_smem + kDqStages * kSubBytes;
  DqBarriers* bars = reinterpret_cast<DqBarriers*>(v_smem + kDqStages * kSubBytes);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // item: a pair of sub-tiles of one (b, kv head); later rows, which see more
  // keys under a staircase, first
  const int bk = blockIdx.x / p.n_pair;
  const int pair = p.n_pair - 1 - (blockIdx.x - bk * p.n_pair);
  const int b = bk / p.Hkv, kvh = bk - b * p.Hkv;
  const int s0 = 2 * pair, n_here = min(2, p.n_sub - s0);
  const int L = kMode == kMaskLength ? length_of(p, b) : 0;

  // first and last position of the pair's rows
  const int mt0 = s0 % p.n_mt, mt1 = (s0 + n_here - 1) % p.n_mt;
  const int m_lo = min(mt0, mt1) * p.MT;
  const int m_hi = min(p.M, (max(mt0, mt1) + 1) * p.MT) - 1;

  // live key chunks [0, a1) and [b0, b1), as in the forward kernel
  int a1 = 0, b0 = 0, b1 = 0;
  if (kMode == kMaskBool) {
    a1 = p.n_chunks;
  } else if (kMode == kMaskLength) {
    a1 = m_lo < L ? (L + kChunk - 1) / kChunk : 0;
  } else {
    a1 = (p.ds + kChunk - 1) / kChunk;
    if (p.de < p.N) {
      const int e2 = max(p.P, min(p.N, p.N - p.M + m_hi + 1));
      b0 = max(p.de / kChunk, a1);
      b1 = (e2 + kChunk - 1) / kChunk;
    }
  }
  const int n_live = a1 + max(0, b1 - b0);
  auto chunk_at = [&](int j) { return j < a1 ? j : b0 + j - a1; };

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int i = 0; i < kDqStages; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->ds_full, 4);
    mbar_init(&bars->staged[0], 2);
    mbar_init(&bars->staged[1], 2);
    mbar_init(&bars->out_full, 1);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == kWarpProducer) {
    // Loads: Q, dO and O of the pair, then the live K/V chunks through a ring.
    int issued = 0;
    if (n_live > 0) {
      mbar_arrive_expect_tx_elect(&bars->q_full,
                                  static_cast<uint32_t>(3 * n_here * p.Gb * p.MT * kRowBytes));
      for (int i = 0; i < n_here; ++i) {
        const int hb = (s0 + i) / p.n_mt, m0 = (s0 + i - hb * p.n_mt) * p.MT;
        const int h = kvh * p.G + hb * p.Gb;
        tma_load_4d_elect(q_smem + i * kSubBytes, &p.tm_q, &bars->q_full, 0, h, m0, b);
        tma_load_4d_elect(do_smem + i * kSubBytes, &p.tm_do, &bars->q_full, 0, h, m0, b);
        tma_load_4d_elect(o_smem + i * kSubBytes, &p.tm_o, &bars->q_full, 0, h, m0, b);
      }
    }
    for (int j = 0; j < n_live; ++j) {
      const int s = j % kDqStages;
      if (!__all_sync(kFullMask, bounded_wait(&bars->k_empty[s], ((j / kDqStages) & 1) ^ 1, abort_flag))) {
        break;
      }
      mbar_arrive_expect_tx_elect(&bars->k_full[s], 2 * kSubBytes);
      tma_load_4d_elect(k_smem + s * kSubBytes, &p.tm_k64, &bars->k_full[s], 0, kvh, chunk_at(j) * kChunk, b);
      tma_load_4d_elect(v_smem + s * kSubBytes, &p.tm_v64, &bars->k_full[s], 0, kvh, chunk_at(j) * kChunk, b);
      issued = j + 1;
    }
    if (n_live > 0) {
      // never leave the CTA with copies in flight (bounded, abort or not)
      bounded_wait(&bars->q_full, 0, abort_flag, false);
      for (int j = max(0, issued - kDqStages); j < issued; ++j)
        bounded_wait(&bars->k_full[j % kDqStages], (j / kDqStages) & 1, abort_flag, false);
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    if (n_live > 0) {
      const uint32_t id_kk = idesc_bf16_f32(128, 64, false), id_kn = idesc_bf16_f32(128, 64, true);
      const uint32_t q0 = smem_u32(q_smem), do0 = smem_u32(do_smem);
      auto issue_scores = [&](int j) {  // S = Q K^T, dP = dO V^T of chunk j
        const int s = j % kDqStages;
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->k_full[s], (j / kDqStages) & 1, abort_flag)))
          return false;
        if (kMode != kMaskBool) {  // K rows that no query sees feed dS K: 0 times NaN
          const int c0 = chunk_at(j) * kChunk;
          const int lo = kMode == kMaskLength ? L - c0 : p.ds - c0;
          const int hi = kMode == kMaskLength ? kChunk : p.de - c0;
          clear_rows(k_smem + s * kSubBytes, max(lo, 0), min(hi, kChunk));
        }
        tc_fence_after();
        const uint32_t k0 = smem_u32(k_smem + s * kSubBytes), v0 = smem_u32(v_smem + s * kSubBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_elect(tmem + kDqS, sdesc_sw128(q0 + 32 * k), sdesc_sw128(k0 + 32 * k), id_kk, k > 0);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_elect(tmem + kDqP, sdesc_sw128(do0 + 32 * k), sdesc_sw128(v0 + 32 * k), id_kk, k > 0);
        umma_commit_elect(&bars->s_full);
        return true;
      };
      bool ok = __all_sync(kFullMask, bounded_wait(&bars->q_full, 0, abort_flag));
      tc_fence_after();
      ok = ok && issue_scores(0);
      for (int j = 0; ok && j < n_live; ++j) {
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->ds_full, j & 1, abort_flag))) break;
        tc_fence_after();
        const int s = j % kDqStages;
        const uint32_t k0 = smem_u32(k_smem + s * kSubBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // dQ += dS K
          umma_ts_elect(tmem + kDqO, tmem + kDqS + 8 * k, sdesc_sw128(k0 + 2048 * k), id_kn,
                        (j > 0 || k > 0) ? 1u : 0u);
        umma_commit_elect(&bars->k_empty[s]);
        if (j + 1 < n_live) {
          ok = issue_scores(j + 1);
        } else {
          umma_commit_elect(&bars->out_full);
        }
      }
      // every issued MMA completes before TMEM is released
      umma_commit_elect(&bars->drain);
      bounded_wait(&bars->drain, 0, abort_flag, false);
    }
    __syncwarp();
  } else {
    // Compute warps: lane quarter w of TMEM, one query row per thread.
    const int half = warp >> 1;  // sub-tile of the pair
    const int st = s0 + half;
    const int row64 = (warp & 1) * 32 + lane;
    const int hb = st / p.n_mt, mt = st - hb * p.n_mt;
    const int m_local = row64 / p.Gb, g = row64 - m_local * p.Gb;
    const int m = mt * p.MT + m_local;
    const bool valid = st < p.n_sub && m_local < p.MT && m < p.M;
    const int h = kvh * p.G + hb * p.Gb + g;
    const long long row = (static_cast<long long>(b) * p.M + m) * p.H + h;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // visible keys [0, rds) U [rde, e2)
    const int rds = kMode == kMaskAnalytic ? p.ds : 0;
    const int rde = kMode == kMaskAnalytic ? p.de : 0;
    const int e2 = kMode == kMaskAnalytic ? max(p.P, min(p.N, p.N - p.M + m + 1))
                   : kMode == kMaskLength ? (m < L ? L : 0) : 0;
    const uint8_t* mrow = nullptr;
    if (kMode == kMaskBool && valid)
      mrow = p.mask + static_cast<long long>(b) * p.mask_sb + static_cast<long long>(m) * p.mask_sm;

    bool ok = true;
    float nl = -INFINITY, nD = 0.f;
    if (n_live > 0) {
      if (valid) {
        const float lse = p.lse[row];
        nl = lse == -INFINITY ? -INFINITY : -lse;  // a row without keys: every P is 0
      }
      ok = __all_sync(kFullMask, bounded_wait(&bars->q_full, 0, abort_flag));
      if (ok && valid && nl != -INFINITY) {
        const uint8_t* dor = do_smem + half * kSubBytes + row64 * kRowBytes;
        const uint8_t* orow = o_smem + half * kSubBytes + row64 * kRowBytes;
        float acc[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          const uint4 a = *reinterpret_cast<const uint4*>(dor + ((v ^ (row64 & 7)) * 16));
          const uint4 o = *reinterpret_cast<const uint4*>(orow + ((v ^ (row64 & 7)) * 16));
          float fa[8], fo[8];
          Elem<__nv_bfloat16>::unpack(a, fa);
          Elem<__nv_bfloat16>::unpack(o, fo);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i & 1] += fa[i] * fo[i];
        }
        nD = -(acc[0] + acc[1]);
      }
    }
    if (st < p.n_sub) {
      float* stat = p.stats + (static_cast<long long>(bk) * p.n_sub + st) * (2 * kSub);
      stat[row64] = nl;
      stat[kSub + row64] = nD;
    }
    const bool warp_active = __any_sync(kFullMask, valid);
    const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
    const uint64_t nl2 = f2_pack(nl, nl), nD2 = f2_pack(nD, nD);
    for (int j = 0; ok && j < n_live; ++j) {
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->s_full, j & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (warp_active) {
        const int c0 = chunk_at(j) * kChunk;
#pragma unroll
        for (int gq = 0; gq < 2; ++gq) {
          const int g0 = c0 + 32 * gq;
          uint32_t vm = 0u;
          if (kMode == kMaskBool) {
            if (mrow != nullptr && g0 < p.N) vm = mask_bits32(mrow, g0, p.N, p.mask_words);
          } else {
            vm = low_bits(rds - g0) | (low_bits(e2 - g0) & ~low_bits(rde - g0));
          }
          const bool full = __all_sync(kFullMask, !valid || vm == 0xffffffffu);
          const bool none = __all_sync(kFullMask, !valid || vm == 0u);
          uint32_t pk[16];
          if (none) {
#pragma unroll
            for (int i = 0; i < 16; ++i) pk[i] = 0u;
          } else {
            float s[32], dp[32];
            tmem_ld32(tbase + kDqS + 32 * gq, s);
            tmem_ld32(tbase + kDqP + 32 * gq, dp);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float x0, x1, d0, d1;
              f2_unpack(f2_fma(f2_pack(s[2 * k], s[2 * k + 1]), sl2, nl2), x0, x1);
              const uint64_t e = f2_pack(ex2(x0), ex2(x1));
              f2_unpack(f2_mul(e, f2_add(f2_pack(dp[2 * k], dp[2 * k + 1]), nD2)), d0, d1);
              if (!full) {
                d0 = (vm >> (2 * k)) & 1u ? d0 : 0.f;
                d1 = (vm >> (2 * k + 1)) & 1u ? d1 : 0.f;
              }
              pk[k] = pack_bf16x2(d0, d1);
            }
          }
          tmem_st16(tbase + kDqS + 16 * gq, pk);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive_elect(&bars->ds_full);
    }
    // Epilogue: scale dQ, stage its rows where O was, one TMA store per
    // sub-tile.
    if (ok && n_live > 0 &&
        !__all_sync(kFullMask, bounded_wait(&bars->out_full, 0, abort_flag)))
      ok = false;
    if (ok && n_live > 0) {
      tc_fence_after();
      if (warp_active) {
        uint8_t* stage = o_smem + half * kSubBytes + row64 * kRowBytes;
#pragma unroll 1
        for (int q4 = 0; q4 < 4; ++q4) {
          float o[16];
          tmem_ld16(tbase + kDqO + 16 * q4, o);
          tmem_wait_ld();
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_bf16x2(o[v * 8 + 2 * e] * p.out_scale, o[v * 8 + 2 * e + 1] * p.out_scale);
            const uint32_t c = static_cast<uint32_t>(2 * q4 + v) ^ static_cast<uint32_t>(row64 & 7);
            st_shared_v4(stage + c * 16, w[0], w[1], w[2], w[3]);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(&bars->staged[half]);
      if ((warp & 1) == 0 && lane == 0 && st < p.n_sub &&
          bounded_wait(&bars->staged[half], 0, abort_flag)) {
        tma_store_4d(&p.tm_dq, o_smem + half * kSubBytes, 0, kvh * p.G + hb * p.Gb, mt * p.MT, b);
        bulk_commit_group();
        bulk_wait_all0();
      }
    } else if (n_live == 0 && valid) {
      uint4* dst = reinterpret_cast<uint4*>(p.dq + row * 64);
#pragma unroll
      for (int v = 0; v < 8; ++v) dst[v] = make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) publish_device_error(p.host_err, VLAK_ERR_DEVICE_TIMEOUT);
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// dkv kernel

struct DkvBarriers {
  uint64_t kv_full, q_full[kDkvStages], q_empty[kDkvStages], s_full, p_full, out_full, staged, drain;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(DkvBarriers) <= kBarrierBytes, "barrier block");

// TMEM columns of the dkv kernel; P^T and dS^T (bf16 pairs) overwrite the
// first halves of S^T and dP^T
constexpr uint32_t kDkvS = 0, kDkvP = 64, kDkvV = 128, kDkvK = 192;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
      ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <int kMode>
__global__ void __launch_bounds__(kThreads, 2) attn_bwd_dkv(const __grid_constant__ BwdParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = aligned_smem(smem_raw);
  uint8_t* k_smem = smem;                       // [128 x 128 B], then the staged dK
  uint8_t* v_smem = k_smem + 2 * kSubBytes;     // then the staged dV
  uint8_t* q_smem = v_smem + 2 * kSubBytes;     // [stage][64 x 128 B]
  uint8_t* do_smem = q_smem + kDkvStages * kSubBytes;
  float* stat_smem = reinterpret_cast<float*>(do_smem + kDkvStages * kSubBytes);  // [stage][128]
  DkvBarriers* bars =
      reinterpret_cast<DkvBarriers*>(reinterpret_cast<uint8_t*>(stat_smem) + kDkvStages * kStatBytes);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int bk = blockIdx.x / p.n_kblk;
  const int k0 = (blockIdx.x - bk * p.n_kblk) * kKeys;
  const int b = bk / p.Hkv, kvh = bk - b * p.Hkv;
  const int L = kMode == kMaskLength ? length_of(p, b) : 0;

  // position blocks [mt_lo, mt_hi) holding a row that sees a key of this CTA
  int mt_lo = 0, mt_hi = p.n_mt;
  if (kMode == kMaskLength) {
    mt_hi = k0 < L ? min(p.n_mt, (L + p.MT - 1) / p.MT) : 0;
  } else if (kMode == kMaskAnalytic) {
    const int pe = min(k0 + kKeys, p.P);  // prefix keys of the CTA: [k0, pe)
    const bool prefix = k0 < min(pe, p.ds) || max(k0, p.de) < pe;
    if (!prefix) {
      const int c = max(k0, p.P);  // the first staircase key: visible from row c - (N - M)
      const int m_first = c - (p.N - p.M);
      mt_lo = c < min(k0 + kKeys, p.N) ? min(p.n_mt, max(0, m_first) / p.MT) : p.n_mt;
    }
  }
  const int per_head = max(0, mt_hi - mt_lo);
  const int n_live = p.n_sub / p.n_mt * per_head;

  if (threadIdx.x == 0) {
    mbar_init(&bars->kv_full, 1);
    for (int i = 0; i < kDkvStages; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
    }
    mbar_init(&bars->s_full, 1);
    mbar_init(&bars->p_full, 4);
    mbar_init(&bars->staged, 4);
    mbar_init(&bars->out_full, 1);
    mbar_init(&bars->drain, 1);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kWarpMma) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  // Rows of the ring that no box covers meet P = dS = 0 in the products; clear
  // them once, so that they are finite.
  {
    const int row0 = p.Gb * p.MT, n = (kSub - row0) * 8;
    for (int i = threadIdx.x; i < 2 * kDkvStages * n; i += kThreads) {
      const int t = i / n;
      reinterpret_cast<uint4*>(q_smem + t * kSubBytes + row0 * kRowBytes)[i - t * n] =
          make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // i-th live sub-tile: head block and position block
  auto sub_at = [&](int i) {
    const int hb = i / per_head;
    return hb * p.n_mt + mt_lo + (i - hb * per_head);
  };

  if (warp == kWarpProducer) {
    int issued = 0;
    if (n_live > 0) {
      mbar_arrive_expect_tx_elect(&bars->kv_full, 4 * kSubBytes);
      tma_load_4d_elect(k_smem, &p.tm_k, &bars->kv_full, 0, kvh, k0, b);
      tma_load_4d_elect(v_smem, &p.tm_v, &bars->kv_full, 0, kvh, k0, b);
    }
    for (int j = 0; j < n_live; ++j) {
      const int s = j % kDkvStages;
      if (!__all_sync(kFullMask, bounded_wait(&bars->q_empty[s], ((j / kDkvStages) & 1) ^ 1, abort_flag))) {
        break;
      }
      const int st = sub_at(j), hb = st / p.n_mt, m0 = (st - hb * p.n_mt) * p.MT;
      const int h = kvh * p.G + hb * p.Gb;
      mbar_arrive_expect_tx_elect(&bars->q_full[s],
                                  static_cast<uint32_t>(2 * p.Gb * p.MT * kRowBytes + kStatBytes));
      tma_load_4d_elect(q_smem + s * kSubBytes, &p.tm_q, &bars->q_full[s], 0, h, m0, b);
      tma_load_4d_elect(do_smem + s * kSubBytes, &p.tm_do, &bars->q_full[s], 0, h, m0, b);
      bulk_load(stat_smem + s * 2 * kSub, p.stats + (static_cast<long long>(bk) * p.n_sub + st) * (2 * kSub),
                kStatBytes, &bars->q_full[s]);
      issued = j + 1;
    }
    if (n_live > 0) {
      bounded_wait(&bars->kv_full, 0, abort_flag, false);
      for (int j = max(0, issued - kDkvStages); j < issued; ++j)
        bounded_wait(&bars->q_full[j % kDkvStages], (j / kDkvStages) & 1, abort_flag, false);
    }
    __syncwarp();
  } else if (warp == kWarpMma) {
    if (n_live > 0) {
      const uint32_t id_kk = idesc_bf16_f32(128, 64, false), id_kn = idesc_bf16_f32(128, 64, true);
      const uint32_t ks = smem_u32(k_smem), vs = smem_u32(v_smem);
      auto issue_scores = [&](int j) {  // S^T = K Q^T, dP^T = V dO^T of sub-tile j
        const int s = j % kDkvStages;
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->q_full[s], (j / kDkvStages) & 1, abort_flag)))
          return false;
        if (kMode == kMaskLength) {  // rows past L meet P = dS = 0: 0 times NaN
          const int st = sub_at(j), m0 = st % p.n_mt * p.MT;
          const int lo = max(0, L - m0) * p.Gb;
          clear_rows(q_smem + s * kSubBytes, lo, kSub);
          clear_rows(do_smem + s * kSubBytes, lo, kSub);
        }
        tc_fence_after();
        const uint32_t q0 = smem_u32(q_smem + s * kSubBytes), do0 = smem_u32(do_smem + s * kSubBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_elect(tmem + kDkvS, sdesc_sw128(ks + 32 * k), sdesc_sw128(q0 + 32 * k), id_kk, k > 0);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_ss_elect(tmem + kDkvP, sdesc_sw128(vs + 32 * k), sdesc_sw128(do0 + 32 * k), id_kk, k > 0);
        umma_commit_elect(&bars->s_full);
        return true;
      };
      bool ok = __all_sync(kFullMask, bounded_wait(&bars->kv_full, 0, abort_flag));
      tc_fence_after();
      ok = ok && issue_scores(0);
      for (int j = 0; ok && j < n_live; ++j) {
        if (!__all_sync(kFullMask, bounded_wait<1>(&bars->p_full, j & 1, abort_flag))) break;
        tc_fence_after();
        const int s = j % kDkvStages;
        const uint32_t q0 = smem_u32(q_smem + s * kSubBytes), do0 = smem_u32(do_smem + s * kSubBytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // dV += P^T dO
          umma_ts_elect(tmem + kDkvV, tmem + kDkvS + 8 * k, sdesc_sw128(do0 + 2048 * k), id_kn,
                        (j > 0 || k > 0) ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k)  // dK += dS^T Q
          umma_ts_elect(tmem + kDkvK, tmem + kDkvP + 8 * k, sdesc_sw128(q0 + 2048 * k), id_kn,
                        (j > 0 || k > 0) ? 1u : 0u);
        umma_commit_elect(&bars->q_empty[s]);
        if (j + 1 < n_live) {
          ok = issue_scores(j + 1);
        } else {
          umma_commit_elect(&bars->out_full);
        }
      }
      umma_commit_elect(&bars->drain);
      bounded_wait(&bars->drain, 0, abort_flag, false);
    }
    __syncwarp();
  } else {
    // Compute warps: one key per thread, a sub-tile's rows along the columns.
    const int key = k0 + warp * 32 + lane;
    const bool valid = key < p.N;
    const uint32_t tbase = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    // rows m in [m_see, m_end) see this key (all of them, none, or from the
    // staircase's step on)
    int m_see = 0, m_end = p.M;
    if (kMode == kMaskAnalytic) {
      if (key >= p.P)
        m_see = key - (p.N - p.M);
      else if (key >= p.ds && key < p.de)
        m_end = 0;
    } else if (kMode == kMaskLength) {
      m_end = key < L ? L : 0;
    }
    if (!valid) m_end = 0;
    const uint64_t sl2 = f2_pack(p.scale_log2, p.scale_log2);
    bool ok = true;
    for (int j = 0; ok && j < n_live; ++j) {
      const int st = sub_at(j), m0 = st % p.n_mt * p.MT, s = j % kDkvStages;
      // columns of the sub-tile that see the key (rows past M or the box carry
      // -lse = -inf, so their P is 0 without a mask)
      uint32_t vm[2];
      if (kMode == kMaskBool) {
        vm[0] = vm[1] = 0u;
        if (valid) {
          const uint8_t* col = p.mask + static_cast<long long>(b) * p.mask_sb + key;
          const uint64_t heads = ~0ull >> (64 - p.Gb);
          const int n = min(p.MT, p.M - m0);
          for (int i = 0; i < n; ++i) {
            if (__ldg(col + static_cast<long long>(m0 + i) * p.mask_sm) == 0) continue;
            const uint64_t bits = heads << (i * p.Gb);
            vm[0] |= static_cast<uint32_t>(bits);
            vm[1] |= static_cast<uint32_t>(bits >> 32);
          }
        }
      } else {
        const int lo = min(max(m_see - m0, 0), kSub) * p.Gb;
        const int hi = min(max(m_end - m0, 0), kSub) * p.Gb;
        const bool last = m_end >= p.M && valid;  // rows past M are masked by their statistics
        vm[0] = ~low_bits(lo) & (last && hi > 0 ? 0xffffffffu : low_bits(hi));
        vm[1] = ~low_bits(lo - 32) & (last && hi > 0 ? 0xffffffffu : low_bits(hi - 32));
      }
      if (!__all_sync(kFullMask, bounded_wait<1>(&bars->q_full[s], (j / kDkvStages) & 1, abort_flag)) ||
          !__all_sync(kFullMask, bounded_wait<1>(&bars->s_full, j & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const float4* stat = reinterpret_cast<const float4*>(stat_smem + s * 2 * kSub);
#pragma unroll
      for (int gq = 0; gq < 2; ++gq) {
        const bool full = __all_sync(kFullMask, !valid || vm[gq] == 0xffffffffu);
        const bool none = __all_sync(kFullMask, vm[gq] == 0u);
        uint32_t pp[16], pd[16];
        if (none) {
#pragma unroll
          for (int i = 0; i < 16; ++i) pp[i] = pd[i] = 0u;
        } else {
          float sv[32], dp[32];
          tmem_ld32(tbase + kDkvS + 32 * gq, sv);
          tmem_ld32(tbase + kDkvP + 32 * gq, dp);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // four rows
            const float4 l4 = stat[8 * gq + i], d4 = stat[16 + 8 * gq + i];
            const uint64_t nl2[2] = {f2_pack(l4.x, l4.y), f2_pack(l4.z, l4.w)};
            const uint64_t nD2[2] = {f2_pack(d4.x, d4.y), f2_pack(d4.z, d4.w)};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int k = 2 * i + u;
              float x0, x1, d0, d1;
              f2_unpack(f2_fma(f2_pack(sv[2 * k], sv[2 * k + 1]), sl2, nl2[u]), x0, x1);
              float e0 = ex2(x0), e1 = ex2(x1);
              f2_unpack(f2_mul(f2_pack(e0, e1),
                               f2_add(f2_pack(dp[2 * k], dp[2 * k + 1]), nD2[u])), d0, d1);
              if (!full) {
                const bool see0 = (vm[gq] >> (2 * k)) & 1u, see1 = (vm[gq] >> (2 * k + 1)) & 1u;
                e0 = see0 ? e0 : 0.f;
                d0 = see0 ? d0 : 0.f;
                e1 = see1 ? e1 : 0.f;
                d1 = see1 ? d1 : 0.f;
              }
              pp[k] = pack_bf16x2(e0, e1);
              pd[k] = pack_bf16x2(d0, d1);
            }
          }
        }
        tmem_st16(tbase + kDkvS + 16 * gq, pp);
        tmem_st16(tbase + kDkvP + 16 * gq, pd);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_elect(&bars->p_full);
    }
    if (ok && n_live > 0 &&
        !__all_sync(kFullMask, bounded_wait(&bars->out_full, 0, abort_flag)))
      ok = false;
    const int row = warp * 32 + lane;
    if (ok && n_live > 0) {
      tc_fence_after();
#pragma unroll 1
      for (int q = 0; q < 8; ++q) {  // dV, then dK, 16 columns at a time
        const float scale = q < 4 ? 1.f : p.out_scale;
        float o[16];
        tmem_ld16(tbase + kDkvV + 16 * q, o);
        tmem_wait_ld();
        uint8_t* stage = (q < 4 ? v_smem : k_smem) + row * kRowBytes;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack_bf16x2(o[v * 8 + 2 * e] * scale, o[v * 8 + 2 * e + 1] * scale);
          const uint32_t c = static_cast<uint32_t>(2 * (q & 3) + v) ^ static_cast<uint32_t>(row & 7);
          st_shared_v4(stage + c * 16, w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      mbar_arrive_elect(&bars->staged);
      if (threadIdx.x == 0 && bounded_wait(&bars->staged, 0, abort_flag)) {
        tma_store_4d(&p.tm_dv, v_smem, 0, kvh, k0, b);
        tma_store_4d(&p.tm_dk, k_smem, 0, kvh, k0, b);
        bulk_commit_group();
        bulk_wait_all0();
      }
    } else if (n_live == 0 && valid) {
      const long long at = ((static_cast<long long>(b) * p.N + key) * p.Hkv + kvh) * 64;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        reinterpret_cast<uint4*>(p.dk + at)[v] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<uint4*>(p.dv + at)[v] = make_uint4(0, 0, 0, 0);
      }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) publish_device_error(p.host_err, VLAK_ERR_DEVICE_TIMEOUT);
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// host

// Sub-tiles: the divisor Gb <= 64 of G whose boxes of Gb heads x MT positions
// need the fewest, the larger one (longer contiguous reads) on a tie.
struct SubTiling {
  int Gb, MT, n_mt, n_sub;
};
SubTiling sub_tiling(int G, int M) {
  SubTiling best{};
  for (int d = 1; d <= std::min(G, kSub); ++d) {
    if (G % d != 0) continue;
    const int mt = std::min(kSub / d, M), n_mt = (M + mt - 1) / mt;
    if (best.Gb == 0 || G / d * n_mt <= best.n_sub) best = SubTiling{d, mt, n_mt, G / d * n_mt};
  }
  return best;
}

int64_t stats_bytes(const vlak_attn_gqa_args* a) {
  const SubTiling t = sub_tiling(static_cast<int>(a->H / a->Hkv), static_cast<int>(a->M));
  return a->B * a->Hkv * t.n_sub * kStatBytes;
}

template <int kMode>
cudaError_t launch_both(const BwdParams& p, unsigned n_dq, unsigned n_dkv, cudaStream_t cs, int device) {
  static std::atomic<int> ready[64];
  if (ready[device].load() == 0) {
    cudaError_t e = cudaFuncSetAttribute(attn_bwd_dq<kMode>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, kDqSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(attn_bwd_dkv<kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kDkvSmem);
    if (e != cudaSuccess) return e;
    ready[device].store(1);
  }
  attn_bwd_dq<kMode><<<n_dq, kThreads, kDqSmem, cs>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || n_dkv == 0) return e;
  attn_bwd_dkv<kMode><<<n_dkv, kThreads, kDkvSmem, cs>>>(p);
  return cudaGetLastError();
}

int bwd_validate(const vlak_attn_train_args* a, int64_t* P, float* scale) {
  if (!a) return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: null arguments");
  int st = vlak_attn_gqa_check(&a->attn, P, scale);
  if (st != VLAK_OK) return st;
  const void* ptrs[4] = {a->grad_o, a->dq, a->dk, a->dv};
  for (const void* ptr : ptrs)
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: pointers must be 16-byte aligned");
  for (int d = 0; d < 3; ++d)
    if (a->grad_o_stride[d] % 8 != 0)
      return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: grad_o strides must be multiples of 8");
  if (reinterpret_cast<uintptr_t>(a->lse) % 4 != 0)
    return set_error(VLAK_ERR_ALIGNMENT, "fused_attention_gqa_bwd: lse must be 4-byte aligned");
  if (a->lengths && a->mask)
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: lengths or a mask, not both");
  if (a->lengths && a->lengths_dtype != VLAK_I32 && a->lengths_dtype != VLAK_I64)
    return set_error(VLAK_ERR_UNSUPPORTED_DTYPE, "lengths must be int32 or int64");
  if (reinterpret_cast<uintptr_t>(a->lengths) % (a->lengths_dtype == VLAK_I64 ? 8 : 4) != 0)
    return set_error(VLAK_ERR_ALIGNMENT, "lengths must be aligned to its element size");
  if (a->mask && (a->mask_stride_b < 0 || a->mask_stride_m < 0))
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "attn_mask strides must be non-negative");
  return VLAK_OK;
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
  if (!workspace || ws_bytes < stats_bytes(a))
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
  p.B = static_cast<int>(a->B);
  p.M = static_cast<int>(a->M);
  p.N = static_cast<int>(a->N);
  p.H = static_cast<int>(a->H);
  p.Hkv = static_cast<int>(a->Hkv);
  p.G = p.H / p.Hkv;
  const SubTiling tl = sub_tiling(p.G, p.M);
  p.Gb = tl.Gb;
  p.MT = tl.MT;
  p.n_mt = tl.n_mt;
  p.n_sub = tl.n_sub;
  p.n_pair = (tl.n_sub + 1) / 2;
  p.n_kblk = (p.N + kKeys - 1) / kKeys;
  p.n_chunks = (p.N + kChunk - 1) / kChunk;
  const int64_t n_dq = a->B * a->Hkv * p.n_pair;
  const int64_t n_dkv = keys_too ? a->B * a->Hkv * p.n_kblk : 0;
  if (n_dq > INT32_MAX || n_dkv > INT32_MAX)
    return set_error(VLAK_ERR_INVALID_ARGUMENT, "fused_attention_gqa_bwd: too many work items");
  p.P = static_cast<int>(P);
  p.ds = static_cast<int>(a->dead_start);
  p.de = static_cast<int>(a->dead_end);
  p.scale_log2 = scale * 1.4426950408889634f;
  // softmax over a single key is constant: its score's gradient is exactly zero
  p.out_scale = p.N == 1 ? 0.f : scale;
  p.host_err = host_error_word(cs);
  p.lse = args.lse;
  p.stats = static_cast<float*>(workspace);
  p.dq = static_cast<__nv_bfloat16*>(args.dq);
  p.dk = static_cast<__nv_bfloat16*>(args.dk);
  p.dv = static_cast<__nv_bfloat16*>(args.dv);
  p.lengths = args.lengths;
  p.lengths_i64 = args.lengths_dtype == VLAK_I64;
  p.mask = static_cast<const uint8_t*>(args.mask);
  p.mask_sb = args.mask_stride_b;
  p.mask_sm = args.mask_stride_m;
  p.mask_words = reinterpret_cast<uintptr_t>(args.mask) % 4 == 0 && args.mask_stride_b % 4 == 0 &&
                 args.mask_stride_m % 4 == 0;

  const uint32_t gb = static_cast<uint32_t>(tl.Gb), mt = static_cast<uint32_t>(tl.MT);
  auto rows = [&](CUtensorMap* m, const void* ptr, const int64_t* s, const char* name) {
    return encode_map(m, ptr, a->H, a->M, a->B, s[2], s[1], s[0], gb, mt, name);
  };
  auto keys = [&](CUtensorMap* m, const void* ptr, const int64_t* s, uint32_t box, const char* name) {
    return encode_map(m, ptr, a->Hkv, a->N, a->B, s[2], s[1], s[0], 1, box, name);
  };
  const int64_t qs[3] = {a->M * a->H * 64, a->H * 64, 64}, ks[3] = {a->N * a->Hkv * 64, a->Hkv * 64, 64};
  st = rows(&p.tm_q, a->q, a->q_stride, "q");
  if (st == VLAK_OK) st = rows(&p.tm_o, a->o, a->o_stride, "o");
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

  const unsigned g_dq = static_cast<unsigned>(n_dq), g_dkv = static_cast<unsigned>(n_dkv);
  cudaError_t e = args.lengths ? launch_both<kMaskLength>(p, g_dq, g_dkv, cs, dev.device)
                  : args.mask  ? launch_both<kMaskBool>(p, g_dq, g_dkv, cs, dev.device)
                               : launch_both<kMaskAnalytic>(p, g_dq, g_dkv, cs, dev.device);
  if (e != cudaSuccess) return set_cuda_error("fused_attention_gqa_bwd launch failed", e);
  return VLAK_OK;
}

}  // namespace

int take_bwd_device_error(int* code) {
  cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(int));
  if (e != cudaSuccess) return set_cuda_error("vlak_device_error_read", e);
  const int zero = 0;
  e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
  if (e != cudaSuccess) return set_cuda_error("vlak_device_error_read", e);
  return VLAK_OK;
}

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
  int st = vlak_attn_gqa_check(&a, nullptr, nullptr);
  if (st != VLAK_OK) return st;
  if (args->attn.B > 0 && args->attn.M > 0 && args->attn.N > 0) *bytes = stats_bytes(&args->attn);
  return VLAK_OK;
}

extern "C" int vlak_attn_gqa_bwd(const vlak_attn_train_args* args, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return vlak::run_bwd(args, workspace, workspace_bytes, stream);
}
