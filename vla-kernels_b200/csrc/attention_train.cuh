// Shared by the training kernels of GQA attention (attention_train_fwd.cu,
// attention_bwd.cu): how queries and keys are cut into items and steps, the
// queue that hands items out, and the issue of tcgen05 products.
//
// Query rows are handled in sub-tiles of up to 64 rows, Gb heads x MT positions
// with Gb a divisor of G, one TMA box each. A row item is two sub-tiles, the 128
// lanes of a TMEM tile, and walks the keys in chunks of 64.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attention_common.cuh"
#include "vlak_device.cuh"
#include "vlak_internal.h"

namespace vlak {
namespace {

constexpr int kMaskAnalytic = 0, kMaskLength = 1, kMaskBool = 2;

constexpr int kSub = 64;                     // rows of a streamed tile
constexpr int kRowBytes = 128;               // 64 bf16
constexpr int kSubBytes = kSub * kRowBytes;  // 8 KB
constexpr int kChunk = 64;                   // keys of a dq step

// Plans are made for a B200's SMs whatever device is current, so that sizes can
// be asked without one and results do not depend on it.
constexpr int kPlanSms = 148;

// Shape, mask and cutting of a call, common to the kernels' parameters.
struct TrainShape {
  int B, M, N, H, Hkv, G;
  int Gb, MT;                         // heads and positions of a sub-tile
  int n_mt, n_hblk, n_sub, n_pair, n_chunks;
  int n_bk;                           // B * Hkv
  int bk_inner;                       // items run over (b, kv head) first
  int P, ds, de;
  float scale, scale_log2;
  int* host_err;
  unsigned* counter;                  // next item
  const void* lengths;
  int lengths_i64;
  // a bool mask, packed: 32 keys of each row [b][key / 32][m], and 32 rows of
  // each key [b][m / 32][key] (see pack_mask)
  uint32_t *row_bits, *col_bits;
  FastDiv by_bk, by_pair, by_hkv, by_mt_count, by_mt, by_gb;
};

__device__ __forceinline__ int length_of(const TrainShape& p, int b) {
  const long long len = p.lengths_i64 ? static_cast<const long long*>(p.lengths)[b]
                                      : static_cast<const int*>(p.lengths)[b];
  return static_cast<int>(min(max(len, 0LL), static_cast<long long>(p.N)));
}

// low n bits set, n clamped to [0, 32]
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : ((1u << n) - 1u);
}

// P and dS as TMEM operands are bf16 pairs packed over the fp32 columns they were
// computed from: half as many, so beside each lies room for what the rounding
// left, again as bf16. In fine calls that is a second operand of the same product,
// which brings P and dS to 16 bits. Without it their rounding is as large as the
// result's own, so errors are sqrt(2) of the least possible, and on rows of few
// keys, where D carries the rounding of P as well, up to 1.7 times. Twice the
// accumulating products cost a long call a third more time; so calls are fine
// whose time goes to launches or to starting and ending items: of at most
// kFineShare steps per SM, or kFineSteps per row item.
constexpr int kFineShare = 8, kFineSteps = 2;

// What a rounded pair leaves, rounded in turn.
__device__ __forceinline__ uint32_t rest_of_pair(float x0, float x1, uint32_t pair) {
  return pack_bf16x2(x0 - __uint_as_float(pair << 16), x1 - __uint_as_float(pair & 0xffff0000u));
}

// 1024-byte aligned start of the dynamic shared memory
__device__ __forceinline__ uint8_t* aligned_smem(uint8_t* raw) {
  return raw + (((smem_u32(raw) + 1023u) & ~1023u) - smem_u32(raw));
}

// Row `row` of sub-tile st of a (b, kv head): position m, head h within the kv
// head, and whether it exists.
struct SubRow {
  int m, g;
  bool valid;
};
__device__ __forceinline__ SubRow sub_row(const TrainShape& p, int st, int row) {
  const int hb = fast_div(st, p.by_mt_count), mt = st - hb * p.n_mt;
  const int local = fast_div(row, p.by_gb);
  SubRow r;
  r.m = mt * p.MT + local;
  r.g = hb * p.Gb + row - local * p.Gb;
  r.valid = st < p.n_sub && local < p.MT && r.m < p.M;
  return r;
}

// Packs a bool mask by rows and, for the backward pass, by keys (32 x 32 per
// warp: a row's word is a ballot, a key's word is the lane's own bits), so that a
// step reads one word per lane. The kernels read each mask byte once per query
// head and pass otherwise: 1835 x 1835, two samples, 6 heads took 349 us forward
// and backward, four times the time without a mask. Bound: HBM, one read.
constexpr int kPackWarps = 8;
__global__ void __launch_bounds__(32 * kPackWarps)
    pack_mask(const uint8_t* mask, long long sb, long long sm, int B, int M, int N, uint32_t* row_bits,
              uint32_t* col_bits) {
  const int lane = threadIdx.x & 31, nw = (N + 31) / 32, mw = (M + 31) / 32;
  const long long tiles = static_cast<long long>(B) * mw * nw;
  for (long long t = blockIdx.x * kPackWarps + (threadIdx.x >> 5); t < tiles;
       t += static_cast<long long>(gridDim.x) * kPackWarps) {
    const int wn = static_cast<int>(t % nw);
    const long long rest = t / nw;
    const int wm = static_cast<int>(rest % mw), b = static_cast<int>(rest / mw);
    const int key = wn * 32 + lane, m0 = wm * 32;
    const uint8_t* at = mask + b * sb + m0 * sm + key;
    uint32_t row = 0u, col = 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const bool on = key < N && m0 + i < M && __ldg(at + i * sm) != 0;
      const uint32_t word = __ballot_sync(kFullMask, on);
      if (lane == i) row = word;
      col |= static_cast<uint32_t>(on) << i;
    }
    if (m0 + lane < M) row_bits[(static_cast<long long>(b) * nw + wn) * M + m0 + lane] = row;
    if (col_bits != nullptr && key < N) col_bits[(static_cast<long long>(b) * mw + wm) * N + key] = col;
  }
}
// the row's bits of keys c to c + 31 (c a multiple of 32 below N)
__device__ __forceinline__ uint32_t row_bits_at(const TrainShape& p, int b, int m, int c) {
  return __ldg(p.row_bits + (static_cast<long long>(b) * ((p.N + 31) / 32) + c / 32) * p.M + m);
}
// the key's bits of positions m to m + 31 (m below M), zero past M
__device__ __forceinline__ uint32_t col_bits_at(const TrainShape& p, int b, int key, int m) {
  const int mw = (p.M + 31) / 32, w = m / 32;
  const uint32_t* at = p.col_bits + (static_cast<long long>(b) * mw + w) * p.N + key;
  return __funnelshift_r(__ldg(at), w + 1 < mw ? __ldg(at + p.N) : 0u, m & 31);
}

// ---------------------------------------------------------------------------
// Items

// An item as the producer hands it out through shared memory (16 bytes at a
// time).
struct __align__(16) Item {
  int live;           // -1: no more items; else its steps
  int dkv, b, kvh;
  int L;              // length of the sample (lengths only)
  int k0;             // dkv: first key
  int s0, n_here;     // dq: first sub-tile and how many (1 or 2)
  int a1, b0;         // dq: live chunks [0, a1) and [b0, ...)
  int mt_lo, mt_hi;   // dkv: live position blocks of each head block
  int j0, part;       // first of the item's steps, where several parts share them
  int pad[2];
};
static_assert(sizeof(Item) == 64, "four vectors");
__device__ __forceinline__ Item load_item(const Item* src) {
  const int4* v = reinterpret_cast<const int4*>(src);
  const int4 x = v[0], y = v[1], z = v[2], w = v[3];
  Item it;
  it.live = x.x; it.dkv = x.y; it.b = x.z; it.kvh = x.w;
  it.L = y.x; it.k0 = y.y; it.s0 = y.z; it.n_here = y.w;
  it.a1 = z.x; it.b0 = z.y; it.mt_lo = z.z; it.mt_hi = z.w;
  it.j0 = w.x; it.part = w.y;
  return it;
}
// Of an item's steps, those of its part: even shares in order.
__device__ __forceinline__ void take_part(Item& it, int part, int parts) {
  const int share = (it.live + parts - 1) / parts;
  it.part = part;
  it.j0 = min(part * share, it.live);
  it.live = min(share, it.live - it.j0);
}

// The steps of an item in order: chunk `pos` (dq), or position block `pos` of
// head block `hb` (dkv).
struct Steps {
  int pos, hb;
  __device__ __forceinline__ void begin(const Item& it) {
    hb = 0;
    pos = it.j0 < it.a1 ? it.j0 : it.j0 - it.a1 + it.b0;
    if (it.dkv) {
      const int per_head = it.mt_hi - it.mt_lo;
      hb = it.j0 > 0 ? it.j0 / per_head : 0;
      pos = it.mt_lo + it.j0 - hb * per_head;
    }
  }
  __device__ __forceinline__ void next(const Item& it) {
    ++pos;
    if (it.dkv) {
      if (pos == it.mt_hi) {
        pos = it.mt_lo;
        ++hb;
      }
    } else if (pos == it.a1) {
      pos = it.b0;
    }
  }
};

// Row item `blk` of a (b, kv head), counted from the last pair of sub-tiles,
// whose rows see the most keys under a staircase: its rows and live chunks.
template <int kMode>
__device__ __forceinline__ void row_item(const TrainShape& p, int blk, Item& it) {
  it.s0 = 2 * (p.n_pair - 1 - blk);
  it.n_here = min(2, p.n_sub - it.s0);
  // first and last position of the rows
  const int s1 = it.s0 + it.n_here - 1;
  const int mt0 = it.s0 - fast_div(it.s0, p.by_mt_count) * p.n_mt;
  const int mt1 = s1 - fast_div(s1, p.by_mt_count) * p.n_mt;
  const int m_lo = min(mt0, mt1) * p.MT;
  const int m_hi = min(p.M, (max(mt0, mt1) + 1) * p.MT) - 1;
  int b1 = 0;
  if (kMode == kMaskBool) {
    it.a1 = p.n_chunks;
  } else if (kMode == kMaskLength) {
    it.a1 = m_lo < it.L ? (it.L + kChunk - 1) / kChunk : 0;
  } else {
    it.a1 = (p.ds + kChunk - 1) / kChunk;
    if (p.de < p.N) {
      const int e2 = max(p.P, min(p.N, p.N - p.M + m_hi + 1));
      it.b0 = max(p.de / kChunk, it.a1);
      b1 = (e2 + kChunk - 1) / kChunk;
    }
  }
  it.live = it.a1 + max(0, b1 - it.b0);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}"
      ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// The four K = 16 products of one 64-deep contraction, from one elected lane.
// Descriptors step by 32 bytes of a swizzled row (SS, both operands) or by 16
// rows of 128 bytes (TS, B).
__device__ __forceinline__ void umma_ss_x4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred e, n, y;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 n, 0, 0;\n\tsetp.eq.b32 y, 0, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, n;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, y;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, y;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, y;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
// A in TMEM at columns x + 0, 16, 32, 48; `acc` 0 starts a new sum; `on` 0
// issues nothing.
__device__ __forceinline__ void umma_ts_x4(uint32_t d, uint32_t x, uint64_t b, uint32_t idesc,
                                           uint32_t acc, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred e, q, p, y;\n\t.reg .b32 x1, x2, x3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.and.b32 q, %5, 0, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 y, 0, 0;\n\t"
      "add.s32 x1, %1, 16;\n\tadd.s32 x2, %1, 32;\n\tadd.s32 x3, %1, 48;\n\t"
      "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x1], b1, %3, y;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x2], b2, %3, y;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x3], b3, %3, y;\n\t}" ::"r"(d),
      "r"(x), "l"(b), "r"(idesc), "r"(acc), "r"(on)
      : "memory");
}
// Two of them: a 32-deep contraction, A at columns x and x + 8.
__device__ __forceinline__ void umma_ts_x2(uint32_t d, uint32_t x, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred e, p, y;\n\t.reg .b32 x1;\n\t.reg .b64 b1;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 y, 0, 0;\n\t"
      "add.s32 x1, %1, 8;\n\tadd.s64 b1, %2, 128;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x1], b1, %3, y;\n\t}" ::"r"(d),
      "r"(x), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// A counter modulo n with the parity of its rounds.
template <int n>
struct Turn {
  uint32_t i = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++i == n) {
      i = 0;
      round ^= 1;
    }
  }
};

// O beyond its bf16 rounding. D = rowsum(dO * O) is a sum in which the bf16
// rounding of O would weigh as much as that of dS where a row's weight lies on
// few keys, so the forward pass keeps the next eight bits of each entry of O: the
// distance of the 32-bit value from its bf16 one, as integers, -2^15 to 2^15,
// rounded to multiples of 2^8, up to 127 of them. So an O that bf16 holds exactly
// (of a row with one key, whose true dS is 0) stays exact, and bytes of zero stand
// for no more bits. Such a row's dS comes out as 8e-8 of D, what the 32-bit sums
// leave; with the upper byte cut off and the lower one's mean added, 1.1e-5.
__device__ __forceinline__ uint32_t low_bytes(const float* x, const uint32_t* hi) {  // of four entries
  int d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t top = i & 1 ? hi[i >> 1] & 0xffff0000u : hi[i >> 1] << 16;
    d[i] = min(static_cast<int>(__float_as_uint(x[i]) - top + 0x80u), 0x7fff);
  }
  // the second byte of each
  return __byte_perm(__byte_perm(d[0], d[1], 0x0051), __byte_perm(d[2], d[3], 0x0051), 0x5410);
}
// the four entries again, from their bf16 values and the word of low_bytes
__device__ __forceinline__ void with_low_bytes(float* x, uint32_t w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // byte i, its sign above it, zero below
    int d;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(d) : "r"(w), "r"(0x0004 | i << 4 | (8 + i) << 8 | (8 + i) << 12));
    x[i] = __int_as_float(__float_as_int(x[i]) + d);
  }
}

// ---------------------------------------------------------------------------
// host

// Sub-tiles: the divisor Gb <= 64 of G whose boxes of Gb heads x MT positions
// need the fewest, the larger one (longer contiguous reads) on a tie.
struct SubTiling {
  int Gb, MT, n_mt, n_sub;
};
inline SubTiling sub_tiling(int G, int M) {
  SubTiling best{};
  for (int d = 1; d <= std::min(G, kSub); ++d) {
    if (G % d != 0) continue;
    const int mt = std::min(kSub / d, M), n_mt = (M + mt - 1) / mt;
    if (best.Gb == 0 || G / d * n_mt <= best.n_sub) best = SubTiling{d, mt, n_mt, G / d * n_mt};
  }
  return best;
}

inline TrainShape train_shape(const vlak_attn_gqa_args* a, int64_t P, float scale, const SubTiling& t) {
  TrainShape s{};
  s.B = static_cast<int>(a->B);
  s.M = static_cast<int>(a->M);
  s.N = static_cast<int>(a->N);
  s.H = static_cast<int>(a->H);
  s.Hkv = static_cast<int>(a->Hkv);
  s.G = s.H / s.Hkv;
  s.Gb = t.Gb;
  s.MT = t.MT;
  s.n_mt = t.n_mt;
  s.n_hblk = t.n_sub / t.n_mt;
  s.n_sub = t.n_sub;
  s.n_pair = (t.n_sub + 1) / 2;
  s.n_chunks = (s.N + kChunk - 1) / kChunk;
  s.n_bk = static_cast<int>(a->B * a->Hkv);
  // Few heads: all their long items first, for balance, their tensors stay in
  // L2. Many: a head's items one after the other, while its tensors are there.
  s.bk_inner = s.n_bk <= 2 * kPlanSms;
  s.P = static_cast<int>(P);
  s.ds = static_cast<int>(a->dead_start);
  s.de = static_cast<int>(a->dead_end);
  // (a positive scale that fp32 rounds to zero: scores of -inf must stay so)
  s.scale = std::max(scale, 0x1p-126f);
  s.scale_log2 = s.scale * 1.4426950408889634f;
  s.by_bk = fast_div_by(static_cast<unsigned>(s.n_bk));
  s.by_pair = fast_div_by(static_cast<unsigned>(s.n_pair));
  s.by_hkv = fast_div_by(static_cast<unsigned>(s.Hkv));
  s.by_mt_count = fast_div_by(static_cast<unsigned>(s.n_mt));
  s.by_mt = fast_div_by(static_cast<unsigned>(s.MT));
  s.by_gb = fast_div_by(static_cast<unsigned>(s.Gb));
  return s;
}
// The inference entry points' checks, and that counts stay within 32 bits: at most
// 2^30 positions or keys (of one head, twice, 275 GB) and 2^34 rows in all (2 TB).
// A sub-tile holds 33 rows or more of a long call, so there are under 2^29.
inline int check_train(const vlak_attn_gqa_args* a, int64_t* P, float* scale, const char* op) {
  const int st = vlak_attn_gqa_check(a, P, scale);
  if (st != VLAK_OK) return st;
  constexpr double kMost = 0x1p34;
  if (a->M > 1 << 30 || a->N > 1 << 30 || static_cast<double>(a->B) * a->M * a->H > kMost ||
      static_cast<double>(a->B) * a->N * a->Hkv > kMost || static_cast<double>(a->B) * a->Hkv > INT32_MAX)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: too many rows or keys", op);
  return VLAK_OK;
}
// The masks of a call beyond the analytic one.
inline int check_train_masks(const vlak_attn_train_args& a, const char* op) {
  if (a.lengths && a.mask)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: lengths or a mask, not both", op);
  if (a.lengths && a.lengths_dtype != VLAK_I32 && a.lengths_dtype != VLAK_I64)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DTYPE, "%s: lengths must be int32 or int64", op);
  if (reinterpret_cast<uintptr_t>(a.lengths) % (a.lengths_dtype == VLAK_I64 ? 8 : 4) != 0)
    return set_errorf(VLAK_ERR_ALIGNMENT, "%s: lengths must be aligned to its element size", op);
  if (a.mask && (a.mask_stride_b < 0 || a.mask_stride_m < 0))
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: attn_mask strides must be non-negative", op);
  return VLAK_OK;
}
inline void set_masks(TrainShape& s, const vlak_attn_train_args& a) {
  s.lengths = a.lengths;
  s.lengths_i64 = a.lengths_dtype == VLAK_I64;
}
// Bytes of the packed mask by rows and by keys, each a multiple of 256.
inline int64_t row_bits_bytes(const vlak_attn_gqa_args& a) {
  return (a.B * ((a.N + 31) / 32) * a.M * 4 + 255) / 256 * 256;
}
inline int64_t col_bits_bytes(const vlak_attn_gqa_args& a) {
  return (a.B * ((a.M + 31) / 32) * a.N * 4 + 255) / 256 * 256;
}
inline cudaError_t launch_pack(const vlak_attn_train_args& a, const TrainShape& s, cudaStream_t cs) {
  const int64_t tiles = a.attn.B * ((a.attn.M + 31) / 32) * ((a.attn.N + 31) / 32);
  const int blocks = static_cast<int>(std::min<int64_t>((tiles + kPackWarps - 1) / kPackWarps, 16 * kPlanSms));
  pack_mask<<<blocks, 32 * kPackWarps, 0, cs>>>(static_cast<const uint8_t*>(a.mask), a.mask_stride_b,
                                                a.mask_stride_m, s.B, s.M, s.N, s.row_bits, s.col_bits);
  return cudaGetLastError();
}
// Whether a call of `total` steps is fine; P, dead keys: as given or resolved.
inline bool fine_call(const vlak_attn_gqa_args& a, int64_t total) {
  const int64_t n_chunks = (a.N + kChunk - 1) / kChunk;
  const int64_t seen = (a.dead_start + kChunk - 1) / kChunk + n_chunks - a.dead_end / kChunk;
  return total <= kFineShare * kPlanSms || std::min(n_chunks, seen) <= kFineSteps;
}
// Parts of an item of `steps` steps, in a call of `total` steps: none longer
// than an SM's even share, but no shorter than eight steps (joining costs
// about that much), and at most 32. And whatever the balance, none longer than
// kMostSteps: some waits last a whole item, a step takes about 0.55 us, and a
// wait gives up after kWaitLimitNs, seven times what that many take.
constexpr int64_t kMostSteps = 1 << 18;
inline int item_parts(int64_t steps, int64_t total) {
  const int64_t most = std::max<int64_t>(8, (total + kPlanSms - 1) / kPlanSms);
  const int64_t balanced = std::min<int64_t>(32, (steps + most - 1) / most);
  return static_cast<int>(std::max<int64_t>({1, balanced, (steps + kMostSteps - 1) / kMostSteps}));
}

}  // namespace
}  // namespace vlak
