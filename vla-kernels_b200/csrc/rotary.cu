// Position rotation of query / key heads, alone or behind a per-head RMS norm
// in the same pass, forward and backward, for sm_100a.
//
// Mathematics. A head of D entries has rd/2 pairs (a, b) that are rotated and
// D - rd entries that pass through. Half layout: pair i is entries
// (i, i + rd/2); interleaved: (2i, 2i + 1). With t = position * f_i
//   y_a = A (u_a cos t - u_b sin t),  y_b = A (u_b cos t + u_a sin t),
// u = x, or u = x * r * w with r = rsqrt(mean(x^2) + eps) (the norm).
// Backward of the rotation is the same with sin negated (a rotation's
// transpose), so it runs the forward kernel. Backward of the norm, with
// g = A R^T dy and hat = x r:
//   dw = sum over rows of g hat,  dx = r (g w - hat * mean(g w hat)).
//
// Angles. position * f_i reaches 10^5..10^9 radians in long contexts, where a
// 32-bit product has lost the fraction of a turn. The product is taken in
// turns (f_i / 2 pi) in 64 bits, its whole turns are removed there, and the
// remaining fraction goes to sincospi in 32 bits. All else is 32-bit: norms,
// dot products and the weight gradient's sums; outputs are rounded once.
//
// Bound: HBM. Each input is read once and each output written once; one angle
// serves every head of its token.
//
// Weight gradients are summed without atomics: a thread keeps its columns'
// sums over all the rows it visits, a block adds its threads in a fixed order
// and writes one partial row, and a second kernel adds the partial rows in a
// fixed order, so results repeat bit for bit.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "vlak_device.cuh"
#include "vlak_internal.h"

namespace vlak {
namespace {

enum { kRotate = 0, kNormFwd = 1, kNormBwd = 2 };

struct RotTensor {
  const void* x;       // (B, M, H, D), strides in elements, entries contiguous
  const void* g;       // gradient of the output (kNormBwd)
  void* y;             // contiguous (B, M, H, D): output, or dx (kNormBwd)
  const void* w;       // (D) norm weight
  float* dw_part;      // [grid.x][D] partial weight gradients (kNormBwd)
  long long x_sb, x_sm, x_sh, g_sb, g_sm, g_sh;
  int H;
};

struct RotParams {
  RotTensor t[2];      // blockIdx.y selects
  const void* pos;
  const double* freq;  // (half) radians per position
  long long tokens;    // B * M
  long long pos_sb, pos_sm;
  int pos_i64, M, D, half, interleaved, w_f32;
  float amp, sign, eps;
  // 16-byte path: log2 of the lanes per head and of the heads side by side
  int lg_units, lg_heads[2];
  int blocks[2];       // blocks of each tensor
};

__device__ __forceinline__ double position_of(const RotParams& p, long long b, long long m) {
  const long long i = b * p.pos_sb + m * p.pos_sm;
  return p.pos_i64 ? static_cast<double>(static_cast<const long long*>(p.pos)[i])
                   : static_cast<double>(static_cast<const int*>(p.pos)[i]);
}

// (A cos t, +-A sin t) of t = pos * f
__device__ __forceinline__ float2 turn_of(const RotParams& p, double pos, double f) {
  const double turns = f * 0.15915494309189533577;  // f / (2 pi)
  const double frac = fma(pos, turns, -rint(pos * turns));
  float s, c;
  sincospif(2.f * static_cast<float>(frac), &s, &c);
  return make_float2(p.amp * c, p.amp * p.sign * s);
}

// the pair turned; one that is not rotated passes through (whatever its mate)
__device__ __forceinline__ float2 turned(float a, float b, float2 cs, bool rotated) {
  return rotated ? make_float2(a * cs.x - b * cs.y, b * cs.x + a * cs.y) : make_float2(a, b);
}

template <typename T>
__device__ __forceinline__ float weight_at(const RotParams& p, const void* w, int d) {
  return p.w_f32 ? static_cast<const float*>(w)[d] : Elem<T>::to_f(static_cast<const T*>(w)[d]);
}

// ---------------------------------------------------------------------------
// One lane per pair: any even D up to 64 K, any alignment. A block of four
// warps takes a token; its warps take the heads in turn. Lane l holds pairs
// l + 32 i, i < K; the entries past rd count as pairs (rd + 2j, rd + 2j + 1)
// that are not rotated.
constexpr int kLaneWarps = 4;

template <typename T, int K, int kMode>
__global__ void __launch_bounds__(32 * kLaneWarps) rotary_lane(const RotParams p) {
  const RotTensor& t = p.t[blockIdx.y];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int pairs = p.D / 2;
  int ia[K], ib[K];
  float wa[K], wb[K], dwa[K], dwb[K];
#pragma unroll
  for (int i = 0; i < K; ++i) {
    const int q = lane + 32 * i;
    const bool there = q < pairs, halves = q < p.half && !p.interleaved;
    ia[i] = !there ? -1 : halves ? q : 2 * q;
    ib[i] = halves ? q + p.half : 2 * q + 1;
    wa[i] = wb[i] = dwa[i] = dwb[i] = 0.f;
    if (kMode != kRotate && there) {
      wa[i] = weight_at<T>(p, t.w, ia[i]);
      wb[i] = weight_at<T>(p, t.w, ib[i]);
    }
  }
  for (long long tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
    const long long b = tok / p.M, m = tok - b * p.M;
    const double pos = position_of(p, b, m);
    float2 cs[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int q = lane + 32 * i;
      cs[i] = q < p.half ? turn_of(p, pos, p.freq[q]) : make_float2(1.f, 0.f);
    }
    for (int h = warp; h < t.H; h += kLaneWarps) {
      const T* x = static_cast<const T*>(t.x) + b * t.x_sb + m * t.x_sm + h * t.x_sh;
      T* y = static_cast<T*>(t.y) + (tok * t.H + h) * p.D;
      float xa[K], xb[K], r = 1.f;
#pragma unroll
      for (int i = 0; i < K; ++i) {
        xa[i] = ia[i] >= 0 ? Elem<T>::to_f(x[ia[i]]) : 0.f;
        xb[i] = ia[i] >= 0 ? Elem<T>::to_f(x[ib[i]]) : 0.f;
      }
      if (kMode != kRotate) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
        r = rsqrtf(warp_sum(ss) / p.D + p.eps);
      }
      if (kMode == kNormBwd) {
        const T* g = static_cast<const T*>(t.g) + b * t.g_sb + m * t.g_sm + h * t.g_sh;
        float ua[K], ub[K], dot = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) {
          const float ga = ia[i] >= 0 ? Elem<T>::to_f(g[ia[i]]) : 0.f;
          const float gb = ia[i] >= 0 ? Elem<T>::to_f(g[ib[i]]) : 0.f;
          const float2 t = turned(ga, gb, cs[i], lane + 32 * i < p.half);
          const float ta = t.x, tb = t.y;
          xa[i] *= r;
          xb[i] *= r;
          dwa[i] += ta * xa[i];
          dwb[i] += tb * xb[i];
          ua[i] = ta * wa[i];
          ub[i] = tb * wb[i];
          dot += ua[i] * xa[i] + ub[i] * xb[i];
        }
        dot = warp_sum(dot) / p.D;
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (ia[i] >= 0) {
            y[ia[i]] = Elem<T>::from_f(r * (ua[i] - xa[i] * dot));
            y[ib[i]] = Elem<T>::from_f(r * (ub[i] - xb[i] * dot));
          }
      } else {
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (ia[i] >= 0) {
            const float ua = kMode == kNormFwd ? xa[i] * r * wa[i] : xa[i];
            const float ub = kMode == kNormFwd ? xb[i] * r * wb[i] : xb[i];
            const float2 t = turned(ua, ub, cs[i], lane + 32 * i < p.half);
            y[ia[i]] = Elem<T>::from_f(t.x);
            y[ib[i]] = Elem<T>::from_f(t.y);
          }
      }
    }
  }
  if (kMode == kNormBwd) {
    __shared__ float part[kLaneWarps][64 * K];
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (ia[i] >= 0) {
        part[warp][ia[i]] = dwa[i];
        part[warp][ib[i]] = dwb[i];
      }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kLaneWarps; ++w) s += part[w][d];
      t.dw_part[static_cast<long long>(blockIdx.x) * p.D + d] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// 16-byte path: a thread holds a unit of two vectors of V entries, the two
// halves of V pairs (half layout), or 2V neighbouring entries (interleaved, and
// past rd). A head is D / 2V units on the next power of two of lanes, so a norm
// is a few shuffles. The 256 threads of a block take `TB` tokens x `HS` heads
// at a time and walk the remaining heads of those tokens, so the angles, which
// the block first computes into shared memory, one sincospi per (token, pair),
// serve every head from registers. Weight-gradient sums stay in registers over
// all the rows a thread visits.
constexpr int kVecThreads = 256;

template <typename T, int kMode>
__global__ void __launch_bounds__(kVecThreads, kMode == kNormBwd ? 2 : 3)
    rotary_vec(const RotParams p) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kRows = kMode == kRotate ? 2 : 1;   // heads in flight per thread
  constexpr int kVecs = kMode == kNormBwd ? 4 : 2;  // vectors per head: x, and the gradient
  // two tables in turn, so one barrier per step is enough: TB * half entries,
  // at most (256 / units) * (units * V)
  __shared__ __align__(16) float2 table[2][kVecThreads * V];
  const int z = static_cast<int>(blockIdx.x) >= p.blocks[0] ? 1 : 0;
  const RotTensor& t = p.t[z];
  const int blk = blockIdx.x - (z ? p.blocks[0] : 0);
  const int u = threadIdx.x & ((1 << p.lg_units) - 1), slot = threadIdx.x >> p.lg_units;
  const int HS = 1 << p.lg_heads[z], h0 = slot & (HS - 1), tl = slot >> p.lg_heads[z];
  const int TB = (kVecThreads >> p.lg_units) >> p.lg_heads[z];
  const int turned_units = p.half / V;
  const bool there = u < p.D / (2 * V), rot = u < turned_units;
  const int e0 = rot ? (p.interleaved ? 2 * u * V : u * V) : 2 * u * V;
  const int e1 = rot && !p.interleaved ? e0 + p.half : e0 + V;
  const unsigned tokens = static_cast<unsigned>(p.tokens), M = p.M;

  float w[2 * V], dw[2 * V];
  if (kMode != kRotate) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[i] = there ? weight_at<T>(p, t.w, e0 + i) : 0.f;
      w[V + i] = there ? weight_at<T>(p, t.w, e1 + i) : 0.f;
      dw[i] = dw[V + i] = 0.f;
    }
  }
  int buf = 0;
  for (unsigned tok0 = blk * TB; tok0 < tokens; tok0 += p.blocks[z] * TB, buf ^= 1) {
    const unsigned tok = tok0 + tl;
    const bool here = there && tok < tokens;
    const long long b = tok / M, m = tok - tok / M * M;
    const T* x = static_cast<const T*>(t.x) + b * t.x_sb + m * t.x_sm;
    const T* g = static_cast<const T*>(t.g) + b * t.g_sb + m * t.g_sm;
    T* y = static_cast<T*>(t.y) + static_cast<long long>(tok) * t.H * p.D;
    uint4 raw[kRows][kVecs];
    auto load = [&](int h) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int hr = h + r * HS;
        if (here && hr < t.H) {
          raw[r][0] = ld_stream16(x + hr * t.x_sh + e0);
          raw[r][1] = ld_stream16(x + hr * t.x_sh + e1);
          if (kMode == kNormBwd) {
            raw[r][kVecs - 2] = ld_stream16(g + hr * t.g_sh + e0);
            raw[r][kVecs - 1] = ld_stream16(g + hr * t.g_sh + e1);
          }
        } else {
#pragma unroll
          for (int v = 0; v < kVecs; ++v) raw[r][v] = make_uint4(0, 0, 0, 0);
        }
      }
    };
    load(h0);  // in flight while the angles are computed
    for (int e = threadIdx.x; e < TB * p.half; e += kVecThreads) {
      const int tt = e / p.half, i = e - tt * p.half;
      const unsigned at = tok0 + tt;
      if (at < tokens)
        table[buf][e] = turn_of(p, position_of(p, at / M, at - at / M * M), p.freq[i]);
    }
    __syncthreads();
    float2 cs[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      cs[i] = rot && here ? table[buf][tl * p.half + u * V + i] : make_float2(1.f, 0.f);
    // turn the unit's pairs (f[0..V) and f[V..2V) are its two vectors)
    auto turn = [&](float (&f)[2 * V]) {
      if (!rot) return;
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 r = turned(f[2 * i], f[2 * i + 1], cs[i], true);
          f[2 * i] = r.x;
          f[2 * i + 1] = r.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 r = turned(f[i], f[V + i], cs[i], true);
          f[i] = r.x;
          f[V + i] = r.y;
        }
      }
    };
    // the sum over the lanes of a head
    auto head_sum = [&](float v) {
      for (int o = (1 << p.lg_units) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
      return v;
    };
    // every lane of a warp makes the same trips (shuffles): up to the block's
    // first head slot
    for (int h = h0; h - h0 < t.H; h += kRows * HS) {
      float f[kRows][2 * V], gr[kMode == kNormBwd ? 2 * V : 1];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        Elem<T>::unpack(raw[r][0], f[r]);
        Elem<T>::unpack(raw[r][1], f[r] + V);
      }
      if constexpr (kMode == kNormBwd) {
        Elem<T>::unpack(raw[0][2], gr);
        Elem<T>::unpack(raw[0][3], gr + V);
      }
      if (h - h0 + kRows * HS < t.H) load(h + kRows * HS);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int hr = h + r * HS;
        float inv = 1.f;
        if (kMode != kRotate) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) ss += f[r][i] * f[r][i];
          inv = rsqrtf(head_sum(ss) / p.D + p.eps);
        }
        if constexpr (kMode == kNormBwd) {
          turn(gr);
          float dot = 0.f;
          const bool row = here && hr < t.H;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            f[r][i] *= inv;
            dw[i] += row ? gr[i] * f[r][i] : 0.f;
            gr[i] *= w[i];
            dot += gr[i] * f[r][i];
          }
          dot = head_sum(dot) / p.D;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) f[r][i] = inv * (gr[i] - f[r][i] * dot);
        } else {
          if (kMode == kNormFwd) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) f[r][i] *= inv * w[i];
          }
          turn(f[r]);
        }
        if (here && hr < t.H) {
          st_stream16(y + hr * p.D + e0, Elem<T>::pack(f[r]));
          st_stream16(y + hr * p.D + e1, Elem<T>::pack(f[r] + V));
        }
      }
    }
  }
  if constexpr (kMode == kNormBwd) {
    // lanes of one unit within the warp, then the warps
#pragma unroll
    for (int i = 0; i < 2 * V; ++i)
      for (int o = 16; o >= (1 << p.lg_units); o >>= 1) dw[i] += __shfl_xor_sync(kFullMask, dw[i], o);
    float* part = reinterpret_cast<float*>(table);  // [warp][D]
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane < (1 << p.lg_units) && there) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        part[warp * p.D + e0 + i] = dw[i];
        part[warp * p.D + e1 + i] = dw[V + i];
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kVecThreads) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kVecThreads / 32; ++k) sum += part[k * p.D + d];
      t.dw_part[static_cast<long long>(blk) * p.D + d] = sum;
    }
  }
}

// dw[d] = sum over the partial rows, in a fixed order: warp y of a block adds
// rows y, y + 32, ..., then the 32 sums are added. blockIdx.y: tensor.
struct DwParams {
  const float* part[2];
  void* dw[2];
  int rows[2];
  int D, w_f32;
};
template <typename T>
__global__ void __launch_bounds__(1024) reduce_dw(const DwParams p) {
  __shared__ float acc[32][33];
  const int z = blockIdx.y, col = threadIdx.x & 31, row0 = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + col;
  float s = 0.f;
  if (d < p.D) {
#pragma unroll 8
    for (int r = row0; r < p.rows[z]; r += 32) s += p.part[z][static_cast<long long>(r) * p.D + d];
  }
  acc[row0][col] = s;
  __syncthreads();
  s = warp_sum(acc[col][row0]);  // warp y now adds column y
  const int dd = blockIdx.x * 32 + row0;
  if (col != 0 || dd >= p.D) return;
  if (p.w_f32)
    static_cast<float*>(p.dw[z])[dd] = s;
  else
    static_cast<T*>(p.dw[z])[dd] = Elem<T>::from_f(s);
}

// ---------------------------------------------------------------------------
constexpr int kMaxHeadDim = 1024;

// Grid of a launch: blocks[i] blocks for tensor i, and the 16-byte path's
// shape if the layout allows it.
struct Launch {
  bool vec;
  int lg_units, lg_heads[2], blocks[2];
};
int lg_ceil(int64_t n) {
  int lg = 0;
  while ((int64_t{1} << lg) < n) ++lg;
  return lg;
}
// The 16-byte path wants whole units (two vectors) in the rotated part and in
// the rest, a head on at most one warp, and vectors on 16-byte boundaries.
bool vectors_fit(const vlak_rotary_args* a, int mode) {
  const int V = a->dtype == VLAK_F32 ? 4 : 8;
  if (a->D % (2 * V) != 0 || a->rotary_dim % (2 * V) != 0 || a->D > 64 * V) return false;
  auto fits = [&](const void* ptr, const int64_t* stride) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && stride[0] % V == 0 && stride[1] % V == 0 &&
           stride[2] % V == 0;
  };
  for (int i = 0; i < a->n_tensors; ++i) {
    const vlak_rotary_tensor& t = a->t[i];
    if (!fits(t.x, t.x_stride) || reinterpret_cast<uintptr_t>(t.y) % 16 != 0) return false;
    if (mode == kNormBwd && !fits(t.grad, t.grad_stride)) return false;
  }
  return true;
}
// Lane path: one block per token, at most sixteen per SM (the rest loop).
int64_t lane_blocks(const vlak_rotary_args* a, int sm_count) {
  return std::min<int64_t>(a->B * a->M, 16ll * sm_count);
}
Launch plan(const vlak_rotary_args* a, int mode, int sm_count) {
  const int64_t tokens = a->B * a->M;
  Launch l{};
  l.vec = vectors_fit(a, mode);
  if (!l.vec) {
    for (int i = 0; i < a->n_tensors; ++i)
      l.blocks[i] = static_cast<int>(lane_blocks(a, sm_count));
    return l;
  }
  l.lg_units = lg_ceil(a->D / (a->dtype == VLAK_F32 ? 8 : 16));
  const int lg_slots = 8 - l.lg_units;
  int64_t heads = 0;
  for (int i = 0; i < a->n_tensors; ++i) heads += a->t[i].H;
  for (int i = 0; i < a->n_tensors; ++i) {
    // four or more heads one after the other on a thread, to spread the angles'
    // and the block's fixed work, but side by side when that leaves SMs idle
    int lg = 0;
    while (a->t[i].H >> (lg + 3) != 0) ++lg;
    lg = std::min(lg, lg_slots);
    auto tiles = [&](int lg_h) { return (tokens + (1 << (lg_slots - lg_h)) - 1) >> (lg_slots - lg_h); };
    while (lg < lg_slots && (int64_t{1} << lg) < a->t[i].H && tiles(lg) < 2 * sm_count) ++lg;
    l.lg_heads[i] = lg;
    // the weights' gradient writes one partial row per block: fewer blocks,
    // shared out by the tensors' heads
    const int64_t most = mode == kNormBwd ? std::max<int64_t>(1, 4ll * sm_count * a->t[i].H / heads)
                                          : 64ll * sm_count;
    l.blocks[i] = static_cast<int>(std::min(tiles(lg), most));
  }
  return l;
}

int validate(const vlak_rotary_args* a, int mode, const char* op) {
  if (!a) return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null arguments", op);
  if (a->dtype != VLAK_F32 && a->dtype != VLAK_F16 && a->dtype != VLAK_BF16)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DTYPE, "%s: heads must be fp32, fp16 or bf16", op);
  if (a->pos_dtype != VLAK_I32 && a->pos_dtype != VLAK_I64)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DTYPE, "%s: positions must be int32 or int64", op);
  if (a->B < 0 || a->M < 0 || a->B > INT32_MAX || a->M > INT32_MAX)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: sizes must be in [0, 2^31)", op);
  if (a->D < 2 || a->D % 2 != 0 || a->D > kMaxHeadDim)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: head_dim must be even, 2 to %d", op, kMaxHeadDim);
  if (a->rotary_dim < 2 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->D)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: the rotated part must be even, 2 to head_dim", op);
  if (a->n_tensors < 1 || a->n_tensors > 2)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: one or two tensors", op);
  if (!isfinite(a->amplitude))
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: amplitude must be finite", op);
  if (mode != kRotate) {
    if (!(a->eps >= 0) || !isfinite(a->eps))
      return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", op);
    if (a->weight_dtype != VLAK_F32 && a->weight_dtype != a->dtype)
      return set_errorf(VLAK_ERR_UNSUPPORTED_DTYPE, "%s: weights must be fp32 or of the heads' dtype", op);
  }
  if (a->B * a->M > INT32_MAX)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: at most 2^31 - 1 tokens", op);
  for (int i = 0; i < a->n_tensors; ++i)
    if (a->t[i].H <= 0 || a->t[i].H > INT32_MAX)
      return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: heads must be positive", op);
  if (a->B * a->M == 0) return VLAK_OK;
  const int esz = a->dtype == VLAK_F32 ? 4 : 2, wsz = a->weight_dtype == VLAK_F32 ? 4 : 2;
  auto off = [](const void* ptr, int size) { return reinterpret_cast<uintptr_t>(ptr) % size != 0; };
  if (!a->positions || !a->inv_freq)
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
  if (off(a->positions, a->pos_dtype == VLAK_I64 ? 8 : 4) || off(a->inv_freq, 8))
    return set_errorf(VLAK_ERR_ALIGNMENT, "%s: pointers must be aligned to their elements", op);
  for (int i = 0; i < a->n_tensors; ++i) {
    const vlak_rotary_tensor& t = a->t[i];
    if (!t.x || !t.y || (mode != kRotate && !t.weight) ||
        (mode == kNormBwd && (!t.grad || !t.grad_weight)))
      return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
    if (off(t.x, esz) || off(t.y, esz) || (mode != kRotate && off(t.weight, wsz)) ||
        (mode == kNormBwd && (off(t.grad, esz) || off(t.grad_weight, wsz))))
      return set_errorf(VLAK_ERR_ALIGNMENT, "%s: pointers must be aligned to their elements", op);
  }
  return VLAK_OK;
}

// Partial weight gradients: what the lane path's grid writes, which is never
// less than the 16-byte path's (so alignment does not enter).
int64_t workspace_bytes(const vlak_rotary_args* a, int sm_count) {
  return a->n_tensors * lane_blocks(a, sm_count) * a->D * 4;
}

template <typename T, int kMode>
cudaError_t launch(const RotParams& p, bool vec, int n, cudaStream_t cs) {
  const dim3 grid(p.blocks[0], n);  // lane path: as many blocks for each tensor
  if (vec)
    rotary_vec<T, kMode><<<p.blocks[0] + p.blocks[1], kVecThreads, 0, cs>>>(p);
  else if (p.D <= 64)
    rotary_lane<T, 1, kMode><<<grid, 32 * kLaneWarps, 0, cs>>>(p);
  else if (p.D <= 128)
    rotary_lane<T, 2, kMode><<<grid, 32 * kLaneWarps, 0, cs>>>(p);
  else if (p.D <= 256)
    rotary_lane<T, 4, kMode><<<grid, 32 * kLaneWarps, 0, cs>>>(p);
  else
    rotary_lane<T, 16, kMode><<<grid, 32 * kLaneWarps, 0, cs>>>(p);
  return cudaGetLastError();
}

template <int kMode>
int run(const vlak_rotary_args* a, void* workspace, int64_t ws_bytes, void* stream, const char* op) {
  clear_error();
  int st = validate(a, kMode, op);
  if (st != VLAK_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (a->B * a->M == 0) {
    if (kMode == kNormBwd) {  // no rows: the weights' gradients are zero
      for (int i = 0; i < a->n_tensors; ++i) {
        if (!a->t[i].grad_weight)
          return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
        const cudaError_t e = cudaMemsetAsync(a->t[i].grad_weight, 0,
                                              a->D * (a->weight_dtype == VLAK_F32 ? 4 : 2), cs);
        if (e != cudaSuccess) return set_cuda_error(op, e);
      }
    }
    return VLAK_OK;
  }
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != VLAK_OK) return st;
  if (dev.cc_major != 10)
    return set_errorf(VLAK_ERR_UNSUPPORTED_DEVICE, "%s: needs an sm_100 device (found sm_%d%d)", op,
                      dev.cc_major, dev.cc_minor);
  const Launch l = plan(a, kMode, dev.sm_count);
  RotParams p{};
  for (int i = 0; i < a->n_tensors; ++i) {
    const vlak_rotary_tensor& t = a->t[i];
    p.t[i] = RotTensor{t.x, t.grad, t.y, t.weight, nullptr,
                       t.x_stride[0], t.x_stride[1], t.x_stride[2],
                       t.grad_stride[0], t.grad_stride[1], t.grad_stride[2],
                       static_cast<int>(t.H)};
    if (kMode == kNormBwd)
      p.t[i].dw_part = static_cast<float*>(workspace) + (i ? static_cast<int64_t>(l.blocks[0]) * a->D : 0);
    p.lg_heads[i] = l.lg_heads[i];
    p.blocks[i] = l.blocks[i];
  }
  if (kMode == kNormBwd) {
    if (!workspace || ws_bytes < workspace_bytes(a, dev.sm_count))
      return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: workspace missing or too small", op);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return set_errorf(VLAK_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", op);
  }
  p.lg_units = l.lg_units;
  p.pos = a->positions;
  p.pos_i64 = a->pos_dtype == VLAK_I64;
  p.pos_sb = a->pos_stride[0];
  p.pos_sm = a->pos_stride[1];
  p.freq = a->inv_freq;
  p.tokens = a->B * a->M;
  p.M = static_cast<int>(a->M);
  p.D = static_cast<int>(a->D);
  p.half = static_cast<int>(a->rotary_dim / 2);
  p.interleaved = a->interleaved != 0;
  p.amp = static_cast<float>(a->amplitude);
  // the backward kernel turns the gradient back, the forward one with the flag
  p.sign = (kMode == kNormBwd) != (a->inverse != 0) ? -1.f : 1.f;
  p.eps = static_cast<float>(a->eps);
  p.w_f32 = a->weight_dtype == VLAK_F32;
  cudaError_t e = a->dtype == VLAK_F32   ? launch<float, kMode>(p, l.vec, a->n_tensors, cs)
                  : a->dtype == VLAK_F16 ? launch<__half, kMode>(p, l.vec, a->n_tensors, cs)
                                         : launch<__nv_bfloat16, kMode>(p, l.vec, a->n_tensors, cs);
  if (e != cudaSuccess) return set_cuda_error(op, e);
  if (kMode == kNormBwd) {
    DwParams d{};
    for (int i = 0; i < a->n_tensors; ++i) {
      d.part[i] = p.t[i].dw_part;
      d.dw[i] = a->t[i].grad_weight;
      d.rows[i] = l.blocks[i];
    }
    d.D = p.D;
    d.w_f32 = p.w_f32;
    const dim3 grid((p.D + 31) / 32, a->n_tensors);
    if (a->dtype == VLAK_F16)
      reduce_dw<__half><<<grid, 1024, 0, cs>>>(d);
    else
      reduce_dw<__nv_bfloat16><<<grid, 1024, 0, cs>>>(d);  // fp32 weights: the type is not used
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(op, e);
  }
  return VLAK_OK;
}

}  // namespace
}  // namespace vlak

extern "C" int vlak_rotary(const vlak_rotary_args* args, void* stream) {
  return vlak::run<vlak::kRotate>(args, nullptr, 0, stream, "rotary");
}

extern "C" int vlak_qk_norm_rotary_fwd(const vlak_rotary_args* args, void* stream) {
  return vlak::run<vlak::kNormFwd>(args, nullptr, 0, stream, "qk_norm_rotary");
}

extern "C" int vlak_qk_norm_rotary_bwd(const vlak_rotary_args* args, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  return vlak::run<vlak::kNormBwd>(args, workspace, workspace_bytes, stream,
                                   "qk_norm_rotary_bwd");
}

extern "C" int vlak_qk_norm_rotary_workspace_size(const vlak_rotary_args* args, int64_t* bytes) {
  using namespace vlak;
  clear_error();
  if (!bytes) return set_error(VLAK_ERR_INVALID_ARGUMENT, "workspace size: null output");
  *bytes = 0;
  int st = validate(args, kNormFwd, "qk_norm_rotary_workspace_size");
  if (st != VLAK_OK) return st;
  if (args->B * args->M == 0) return VLAK_OK;
  DeviceInfo dev;
  st = current_device_info(&dev);
  if (st != VLAK_OK) return st;
  *bytes = workspace_bytes(args, dev.sm_count);
  return VLAK_OK;
}
