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
// 32-bit product has lost the fraction of a turn. Whole turns do not matter, so
// f_i / 2 pi is held as a 64-bit binary fraction of a turn and the product with
// the position wraps modulo 2^64, exactly: of what is left the upper 32 bits,
// the fraction of a turn to 2^-32, go to a 32-bit sine and cosine. All else is 32-bit
// too: norms, dot products and the weight gradient's sums; outputs are rounded
// once.
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
  // 16-byte path: log2 of the lanes per head, a block's tokens, the slots of
  // each token that serve queries and keys, and the heads a slot takes in turn
  int lg_units, block_tokens, q_slots, k_slots, trips;
  FastDiv by_M;
};

__device__ __forceinline__ unsigned long long position_of(const RotParams& p, long long b, long long m) {
  const long long i = b * p.pos_sb + m * p.pos_sm;
  return p.pos_i64 ? static_cast<const long long*>(p.pos)[i] : static_cast<const int*>(p.pos)[i];
}

// f radians as a fraction of a turn, modulo whole turns, in units of 2^-64
__device__ __forceinline__ unsigned long long turns_of(double f) {
  const double turns = f * 0.15915494309189533577;  // f / 2 pi
  return __double2ull_rd((turns - floor(turns)) * 0x1p63) << 1;
}
// (A cos t, +-A sin t) of the turn position * turns. For 16-bit heads the
// hardware's sine and cosine: within 2^-21 of the value on half a turn to each
// side, 2^-10 of half a step of fp16, beside which the 2^-26 of a turn that a float
// of the fraction may be off (9e-8 radians) are nothing. For 32-bit heads sincospi,
// four times the instructions, and what the float left of the fraction, r, by
// cos (t + r) = cos t - r sin t, sin (t + r) = sin t + r cos t: without it results
// were 1.33 times as far off as with angles in 64 bits, with it 0.98 times, in the
// same time (8191 x 40 heads of 128: 54 us).
template <typename T>
__device__ __forceinline__ float2 turn_of(const RotParams& p, unsigned long long pos,
                                          unsigned long long turns) {
  const int part = static_cast<int>((pos * turns) >> 32);  // of a turn, in 2^-32, -1/2 to 1/2
  constexpr float kRadians = 1.4629180792671596e-9f;       // 2 pi 2^-32
  const float near = static_cast<float>(part);
  float s, c;
  if constexpr (sizeof(T) == 2) {
    __sincosf(near * kRadians, &s, &c);
  } else {
    float s0, c0;
    sincospif(near * 0x1p-31f, &s0, &c0);
    const float r = static_cast<float>(part - __float2int_rn(near)) * kRadians;
    c = fmaf(-r, s0, c0);
    s = fmaf(r, c0, s0);
  }
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
  // Heads of up to 256 entries: frequencies in registers, and the next head's
  // entries are loaded before this one's work (9 x 954 x 24 heads of 72, rotation
  // forward and backward: 75 -> 68 us). Bound: issue, of loads of single entries.
  constexpr bool kAhead = K <= 4;
  unsigned long long turns[kAhead ? K : 1];
  if constexpr (kAhead) {
#pragma unroll
    for (int i = 0; i < K; ++i) turns[i] = lane + 32 * i < p.half ? turns_of(p.freq[lane + 32 * i]) : 0;
  }
  for (long long tok = blockIdx.x; tok < p.tokens; tok += gridDim.x) {
    const long long b = tok / p.M, m = tok - b * p.M;
    T na[K], nb[K], ma[K], mb[K];  // entries of x, and of the gradient
    auto fetch = [&](int h) {
      if (h >= t.H) return;
      const T* x = static_cast<const T*>(t.x) + b * t.x_sb + m * t.x_sm + h * t.x_sh;
      const T* g = static_cast<const T*>(t.g) + b * t.g_sb + m * t.g_sm + h * t.g_sh;
#pragma unroll
      for (int i = 0; i < K; ++i)
        if (ia[i] >= 0) {
          na[i] = x[ia[i]];
          nb[i] = x[ib[i]];
          if (kMode == kNormBwd) {
            ma[i] = g[ia[i]];
            mb[i] = g[ib[i]];
          }
        }
    };
    if (kAhead) fetch(warp);
    const unsigned long long pos = position_of(p, b, m);
    float2 cs[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int q = lane + 32 * i;
      cs[i] = make_float2(1.f, 0.f);
      if (q < p.half) {
        if constexpr (kAhead)
          cs[i] = turn_of<T>(p, pos, turns[i]);
        else
          cs[i] = turn_of<T>(p, pos, turns_of(p.freq[q]));
      }
    }
    for (int h = warp; h < t.H; h += kLaneWarps) {
      T* y = static_cast<T*>(t.y) + (tok * t.H + h) * p.D;
      float xa[K], xb[K], gx[K], gy[K], r = 1.f;
      if (!kAhead) fetch(h);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        xa[i] = ia[i] >= 0 ? Elem<T>::to_f(na[i]) : 0.f;
        xb[i] = ia[i] >= 0 ? Elem<T>::to_f(nb[i]) : 0.f;
        if (kMode == kNormBwd) {
          gx[i] = ia[i] >= 0 ? Elem<T>::to_f(ma[i]) : 0.f;
          gy[i] = ia[i] >= 0 ? Elem<T>::to_f(mb[i]) : 0.f;
        }
      }
      if (kAhead) fetch(h + kLaneWarps);
      if (kMode != kRotate) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) ss += xa[i] * xa[i] + xb[i] * xb[i];
        r = rsqrtf(warp_sum(ss) / p.D + p.eps);
      }
      if (kMode == kNormBwd) {
        float ua[K], ub[K], dot = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) {
          const float2 t = turned(gx[i], gy[i], cs[i], lane + 32 * i < p.half);
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
// 16-byte path: a thread holds a unit of two vectors of V entries, one from each
// half of the rotated part, or of the part past rd, in both layouts: in the half
// layout they are the halves of V pairs, in the interleaved one V / 2 pairs each.
// So a head's lanes read neighbouring 16 bytes. A head is D / 2V units on the next
// power of two of lanes, a slot, so a norm is a few shuffles. A block takes TB tokens at a time with HS slots
// each; some of the HS serve queries and the others keys, in turn over their
// heads, so a thread stays with one tensor and its weight-gradient sums stay in
// registers. The block first computes the tokens' angles into shared memory,
// once for all heads of queries and keys.
constexpr int kVecThreads = 128;
// Blocks per SM, by registers.
constexpr int vec_blocks(int mode) { return mode == kRotate ? 6 : mode == kNormFwd ? 5 : 4; }

// Arithmetic is on pairs of fp32 (f32x2), which halves its issue slots; the
// forward norm folds its weights into the angles' factors once per token:
//   y_a = r (x_a c w_a - x_b s w_b),  y_b = r (x_b c w_b + x_a s w_a).
// A unit's 2V entries are held as V entries a and their V mates b; the
// interleaved layout is taken apart while unpacking, which costs nothing, so
// both layouts share all arithmetic.
template <typename T, bool kInter>
__device__ __forceinline__ void unpack_unit(const uint4& v0, const uint4& v1, uint64_t* f) {
  constexpr int V = Elem<T>::kVec;
  float t[2 * V];
  Elem<T>::unpack(v0, t);
  Elem<T>::unpack(v1, t + V);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    f[i] = kInter ? f2_pack(t[4 * i], t[4 * i + 2]) : f2_pack(t[2 * i], t[2 * i + 1]);
    f[V / 2 + i] = kInter ? f2_pack(t[4 * i + 1], t[4 * i + 3]) : f2_pack(t[V + 2 * i], t[V + 2 * i + 1]);
  }
}
template <typename T, bool kInter>
__device__ __forceinline__ void pack_unit(const uint64_t* f, uint4& v0, uint4& v1) {
  constexpr int V = Elem<T>::kVec;
  float t[2 * V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if (kInter) {
      f2_unpack(f[i], t[4 * i], t[4 * i + 2]);
      f2_unpack(f[V / 2 + i], t[4 * i + 1], t[4 * i + 3]);
    } else {
      f2_unpack(f[i], t[2 * i], t[2 * i + 1]);
      f2_unpack(f[V / 2 + i], t[V + 2 * i], t[V + 2 * i + 1]);
    }
  }
  v0 = Elem<T>::pack(t);
  v1 = Elem<T>::pack(t + V);
}

// Rows come through shared memory, kDepth - 1 ahead of the one being worked on: a
// thread's own vectors, so without barriers. One row ahead in registers left the
// kernels waiting for loads: 2 x 8192 tokens of 40 heads of 128 took 60.4 us
// instead of 53.2, 8191 tokens with norm 36.2 instead of 31.0 forward, 60 instead
// of 51 backward; the depth (2 to 4) hardly matters. These copies go past L1, so a
// warp's have to cover whole sectors (see the units above; 76 us with
// neighbouring vectors per thread).
__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

template <typename T, int kMode, bool kInter>
__global__ void __launch_bounds__(kVecThreads, vec_blocks(kMode))
    rotary_vec(const RotParams p) {
  constexpr int V = Elem<T>::kVec;
  constexpr int kDepth = kMode == kNormBwd ? 3 : 4, kVecs = kMode == kNormBwd ? 4 : 2;
  __shared__ uint4 ring[kDepth][kVecs][kVecThreads];
  // two tables in turn, so one barrier per step is enough: TB * half entries,
  // at most slots * (units * V). Tables lie as [chunk of 16 bytes][unit], so that
  // a warp's units read neighbouring 16 bytes.
  __shared__ __align__(16) float2 table[2][kVecThreads * V];
  __shared__ __align__(16) float w_smem[2][kMode != kRotate ? 64 * V : 4];  // [chunk][32 units][4]
  const int u = threadIdx.x & ((1 << p.lg_units) - 1), slot = threadIdx.x >> p.lg_units;
  const int HS = p.q_slots + p.k_slots, TB = p.block_tokens;
  const int tl = slot / HS, hs = slot - tl * HS;  // token and place of the slot
  const bool z = hs >= p.q_slots;                 // a key slot
  const RotTensor& t = z ? p.t[1] : p.t[0];
  const int H = t.H, h0 = z ? hs - p.q_slots : hs, h_step = z ? p.k_slots : p.q_slots;
  const unsigned stride = gridDim.x * TB;
  const int units = p.D / (2 * V), turned_units = max(1, p.half / V);
  const bool there = u < units, rot = u < p.half / V;
  // the unit's vectors start at entries e0 and e0 + apart
  const int past = p.D / 2 - p.half;  // half of the entries past rd
  const int e0 = !there ? 0 : rot ? u * V : p.half + u * V;
  const int apart = rot || !there ? p.half : past;
  auto entry = [&](int i) {  // of the i-th a (i < V) or b
    const int k = i % V;
    return kInter ? e0 + (k < V / 2 ? 2 * k : apart + 2 * k - V) + i / V : e0 + k + (i < V ? 0 : apart);
  };
  const unsigned tokens = static_cast<unsigned>(p.tokens);
  const float inv_D = 1.f / p.D;
  const long long x_step = h_step * t.x_sh, g_step = h_step * t.g_sh;
  const int y_step = h_step * p.D;
  // A thread fills table entries (token, pair) 256 apart; the pair stays the
  // same, and its frequency in a register, when it can.
  const int step_tok = kVecThreads / p.half, step_pair = kVecThreads - step_tok * p.half;
  const int fill_tok = threadIdx.x / p.half, fill_pair = threadIdx.x - fill_tok * p.half;
  unsigned long long fill_turns = 0;

  uint64_t dw[kMode == kNormBwd ? V : 1];
  if (kMode == kNormBwd) {
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = 0ull;
  }
  // the 2i-th and (2i + 1)-th pairs of the unit's weights
  auto w_pairs = [&](int i, uint64_t& a, uint64_t& c) {
    const float4 w = *reinterpret_cast<const float4*>(&w_smem[z][(i * 32 + u) * 4]);
    a = f2_pack(w.x, w.y);
    c = f2_pack(w.z, w.w);
  };
  // the next row to fetch: of tile l_tok0 the head l_h, in the l_trip-th trip. A
  // thread without one (no token, head or unit) works on what the ring holds; its
  // results go nowhere.
  unsigned l_tok0 = blockIdx.x * TB;
  int l_trip = 0, l_h = h0;
  bool l_here = false;
  const T *l_x = nullptr, *l_g = nullptr;
  auto locate = [&]() {
    const unsigned tok = l_tok0 + tl;
    l_here = there && tl < TB && tok < tokens;
    if (l_here) {
      const unsigned tb = fast_div(tok, p.by_M);
      const long long b = tb, m = tok - tb * p.by_M.d;
      l_x = static_cast<const T*>(t.x) + b * t.x_sb + m * t.x_sm + h0 * t.x_sh + e0;
      if (kMode == kNormBwd) l_g = static_cast<const T*>(t.g) + b * t.g_sb + m * t.g_sm + h0 * t.g_sh + e0;
    }
  };
  auto fetch = [&](int to) {
    if (l_here && l_h < H) {
      copy16_async(&ring[to][0][threadIdx.x], l_x);
      copy16_async(&ring[to][1][threadIdx.x], l_x + apart);
      if (kMode == kNormBwd) {
        copy16_async(&ring[to][2][threadIdx.x], l_g);
        copy16_async(&ring[to][3][threadIdx.x], l_g + apart);
      }
    }
    copies_commit();
    l_x += x_step;
    if (kMode == kNormBwd) l_g += g_step;
    l_h += h_step;
    if (++l_trip == p.trips) {
      l_trip = 0;
      l_h = h0;
      l_tok0 += stride;
      locate();
    }
  };
  locate();
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  int at_ring = 0;
  bool first = true;
  int buf = 0;
  for (unsigned tok0 = blockIdx.x * TB; tok0 < tokens; tok0 += stride, buf ^= 1) {
    const bool here = there && tl < TB && tok0 + tl < tokens;
    const unsigned tok = tl < TB && tok0 + tl < tokens ? tok0 + tl : tok0;
    T* y = static_cast<T*>(t.y) + (static_cast<long long>(tok) * H + h0) * p.D + e0;
    if (first) {
      first = false;
      fill_turns = turns_of(p.freq[fill_pair]);
      if (kMode != kRotate) {
        for (int e = threadIdx.x; e < p.D; e += kVecThreads) {
          // entry e as the i-th a or b of its unit: c-th of the first or second
          // half of its part
          const bool turns = e < 2 * p.half;
          const int len = turns ? p.half : past, from = turns ? 0 : 2 * p.half;
          const int second = e - from >= len, c = e - from - second * len;
          const int eu = (turns ? 0 : p.half / V) + c / V, r = c % V;
          const int i = kInter ? second * (V / 2) + r / 2 + r % 2 * V : r + second * V;
          const int at = ((i / 4) * 32 + eu) * 4 + i % 4;
          w_smem[0][at] = weight_at<T>(p, p.t[0].w, e);
          if (p.k_slots) w_smem[1][at] = weight_at<T>(p, p.t[1].w, e);
        }
      }
    }
    for (int tt = fill_tok, i = fill_pair; tt < TB;) {
      const unsigned at = tok0 + tt;
      if (at < tokens) {
        const unsigned ab = fast_div(at, p.by_M);
        const unsigned long long turns = step_pair == 0 ? fill_turns : turns_of(p.freq[i]);
        // pair i is the j-th of unit `unit`
        int unit = i / V, j = i % V;
        if (kInter) {
          const int vec = i / (V / 2), second = vec >= turned_units;
          unit = vec - second * turned_units;
          j = second * (V / 2) + i % (V / 2);
        }
        table[buf][((tt * (V / 2) + j / 2) * turned_units + unit) * 2 + j % 2] =
            turn_of<T>(p, position_of(p, ab, at - ab * p.by_M.d), turns);
      }
      tt += step_tok;
      i += step_pair;
      if (i >= p.half) {
        i -= p.half;
        ++tt;
      }
    }
    __syncthreads();
    // Factors: y_a = Ca a + Sa b, y_b = Cb b + Sb a, in pairs; Ca and Cb are
    // one unless weights are folded in.
    constexpr int kC = kMode == kNormFwd ? V : V / 2;
    uint64_t C[kC], S[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float4 cs = make_float4(1.f, 0.f, 1.f, 0.f);
      if (rot && here)
        cs = *reinterpret_cast<const float4*>(&table[buf][((tl * (V / 2) + i) * turned_units + u) * 2]);
      C[i] = f2_pack(cs.x, cs.z);
      S[i] = f2_pack(-cs.y, -cs.w);
      S[V / 2 + i] = f2_pack(cs.y, cs.w);
    }
    if constexpr (kMode == kNormFwd) {
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        uint64_t wa[2], wb[2];
        w_pairs(i, wa[0], wa[1]);
        w_pairs(V / 4 + i, wb[0], wb[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = 2 * i + j;
          C[V / 2 + k] = f2_mul(C[k], wb[j]);
          C[k] = f2_mul(C[k], wa[j]);
          S[k] = f2_mul(S[k], wb[j]);
          S[V / 2 + k] = f2_mul(S[V / 2 + k], wa[j]);
        }
      }
    }
    auto turn = [&](uint64_t (&f)[V]) {
      if (!rot) {  // passes through, whatever its neighbour
        if constexpr (kMode == kNormFwd) {
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = f2_mul(f[i], C[i]);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const uint64_t a = f[i], c = f[V / 2 + i];
        f[i] = f2_fma(c, S[i], f2_mul(a, C[i]));
        f[V / 2 + i] = f2_fma(a, S[V / 2 + i], f2_mul(c, C[(V / 2 + i) % kC]));
      }
    };
    // the sum over the lanes of a head
    auto head_sum = [&](uint64_t v2) {
      float lo, hi;
      f2_unpack(v2, lo, hi);
      float v = lo + hi;
#pragma unroll
      for (int k = 0; k < 5; ++k)
        if (k < p.lg_units) v += __shfl_xor_sync(kFullMask, v, 1 << k);
      return v;
    };
    // every lane makes the same trips (shuffles)
    for (int k = 0, h = h0; k < p.trips; ++k, h += h_step) {
      const bool row = here && h < H;
      uint64_t f[V], gr[kMode == kNormBwd ? V : 1];
      fetch(at_ring == 0 ? kDepth - 1 : at_ring - 1);
      copies_wait<kDepth - 1>();
      unpack_unit<T, kInter>(ring[at_ring][0][threadIdx.x], ring[at_ring][1][threadIdx.x], f);
      if constexpr (kMode == kNormBwd)
        unpack_unit<T, kInter>(ring[at_ring][2][threadIdx.x], ring[at_ring][3][threadIdx.x], gr);
      at_ring = at_ring == kDepth - 1 ? 0 : at_ring + 1;
      if constexpr (kMode == kNormBwd) {
        // with u = w R^T g, both sums in one round of shuffles:
        //   dx = r (u - x r^2 sum(u x) / D),  dw += (R^T g) (x r)
        turn(gr);
        uint64_t ss[2] = {0ull, 0ull}, ux[2] = {0ull, 0ull}, un[V];
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          uint64_t wa, wb;
          w_pairs(i / 2, wa, wb);
          un[i] = f2_mul(gr[i], wa);
          un[i + 1] = f2_mul(gr[i + 1], wb);
          ss[0] = f2_fma(f[i], f[i], ss[0]);
          ss[1] = f2_fma(f[i + 1], f[i + 1], ss[1]);
          ux[0] = f2_fma(un[i], f[i], ux[0]);
          ux[1] = f2_fma(un[i + 1], f[i + 1], ux[1]);
        }
        if (!there) ss[0] = ss[1] = ux[0] = ux[1] = 0ull;
        const float sum_xx = head_sum(f2_add(ss[0], ss[1])), sum_ux = head_sum(f2_add(ux[0], ux[1]));
        const float inv = rsqrtf(fmaf(sum_xx, inv_D, p.eps)), nd = -inv * inv * (sum_ux * inv_D);
        const uint64_t inv2 = f2_pack(inv, inv), nd2 = f2_pack(nd, nd);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (row) dw[i] = f2_fma(f2_mul(gr[i], inv2), f[i], dw[i]);
          f[i] = f2_mul(f2_fma(f[i], nd2, un[i]), inv2);
        }
      } else {
        if constexpr (kMode == kNormFwd) {
          uint64_t ss[2] = {0ull, 0ull};
#pragma unroll
          for (int i = 0; i < V; ++i) ss[i & 1] = f2_fma(f[i], f[i], ss[i & 1]);
          if (!there) ss[0] = ss[1] = 0ull;
          const float inv = rsqrtf(fmaf(head_sum(f2_add(ss[0], ss[1])), inv_D, p.eps));
          const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = f2_mul(f[i], inv2);
        }
        turn(f);
      }
      if (row) {
        uint4 v0, v1;
        pack_unit<T, kInter>(f, v0, v1);
        st_stream16(y, v0);
        st_stream16(y + apart, v1);
      }
      y += y_step;
    }
  }
  if constexpr (kMode == kNormBwd) {
    // one sum per tensor over the slots, in their order
    float* part = reinterpret_cast<float*>(table);  // [slot][D]
    __syncthreads();
    if (there) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float lo, hi;
        f2_unpack(dw[i], lo, hi);
        part[slot * p.D + entry(2 * i)] = lo;
        part[slot * p.D + entry(2 * i + 1)] = hi;
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * p.D; e += kVecThreads) {
      const int zz = e >= p.D, d = e - zz * p.D;
      if (zz && p.k_slots == 0) break;
      float sum = 0.f;
      for (int tt = 0; tt < TB; ++tt)
        for (int q = zz ? p.q_slots : 0; q < (zz ? HS : p.q_slots); ++q)
          sum += part[(tt * HS + q) * p.D + d];
      p.t[zz].dw_part[static_cast<long long>(blockIdx.x) * p.D + d] = sum;
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

// Grid of a launch, and the 16-byte path's shape if the layout allows it.
struct Launch {
  bool vec;
  int blocks, lg_units, block_tokens, q_slots, k_slots, trips;
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
    l.blocks = static_cast<int>(lane_blocks(a, sm_count));
    return l;
  }
  l.lg_units = lg_ceil(a->D / (a->dtype == VLAK_F32 ? 8 : 16));
  const int64_t slots = kVecThreads >> l.lg_units, Hq = a->t[0].H;
  const int64_t Hk = a->n_tensors > 1 ? a->t[1].H : 0;
  // Trips over the heads: a slot's cost per token is its trips plus about one
  // trip's worth of fixed work, times the slots a token takes (unused ones
  // included); the cheapest, but with more slots side by side while the tokens
  // leave SMs without a block.
  double best = 0;
  for (int64_t trips = 1; trips <= std::max(Hq, Hk); ++trips) {
    const int64_t q = (Hq + trips - 1) / trips, k = (Hk + trips - 1) / trips;
    const int64_t tokens_here = slots / (q + k);
    if (tokens_here == 0) continue;
    const double cost = static_cast<double>(trips + 1) * slots / tokens_here;
    const bool spread = (tokens + tokens_here - 1) / tokens_here >= 2 * sm_count;
    if (best == 0 || (spread && cost < best)) {
      best = cost;
      l.block_tokens = static_cast<int>(tokens_here);
      l.q_slots = static_cast<int>(q);
      l.k_slots = static_cast<int>(k);
      l.trips = static_cast<int>(trips);
    }
    if (!spread || trips >= 16) break;
  }
  const int64_t tiles = (tokens + l.block_tokens - 1) / l.block_tokens;
  // Blocks: for the norm as many as are resident, which go over their tiles with
  // rows of the next one in flight, and lay out their weights, and write a partial
  // weight gradient, once. For the rotation alone a tile each, up to 64 per SM:
  // 2 x 8192 tokens of 40 heads of 128 in 53 us, against 63 by resident blocks.
  l.blocks = static_cast<int>(std::min<int64_t>(tiles, (mode == kRotate ? 64ll : vec_blocks(mode)) * sm_count));
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
  // (both as the kernels take them, in 32 bits)
  if (!isfinite(static_cast<float>(a->amplitude)))
    return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: amplitude must be finite", op);
  if (mode != kRotate) {
    if (!(a->eps >= 0) || !isfinite(static_cast<float>(a->eps)))
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
cudaError_t launch(const RotParams& p, bool vec, int blocks, int n, cudaStream_t cs) {
  const dim3 grid(blocks, n);
  if (vec)
    p.interleaved ? rotary_vec<T, kMode, true><<<blocks, kVecThreads, 0, cs>>>(p)
                  : rotary_vec<T, kMode, false><<<blocks, kVecThreads, 0, cs>>>(p);
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
      p.t[i].dw_part = static_cast<float*>(workspace) + static_cast<int64_t>(i) * l.blocks * a->D;
  }
  if (kMode == kNormBwd) {
    if (!workspace || ws_bytes < workspace_bytes(a, dev.sm_count))
      return set_errorf(VLAK_ERR_INVALID_ARGUMENT, "%s: workspace missing or too small", op);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
      return set_errorf(VLAK_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", op);
  }
  p.lg_units = l.lg_units;
  p.block_tokens = l.block_tokens;
  p.q_slots = l.q_slots;
  p.k_slots = l.k_slots;
  p.trips = l.trips;
  p.pos = a->positions;
  p.pos_i64 = a->pos_dtype == VLAK_I64;
  p.pos_sb = a->pos_stride[0];
  p.pos_sm = a->pos_stride[1];
  p.freq = a->inv_freq;
  p.tokens = a->B * a->M;
  p.M = static_cast<int>(a->M);
  p.by_M = fast_div_by(static_cast<unsigned>(a->M));
  p.D = static_cast<int>(a->D);
  p.half = static_cast<int>(a->rotary_dim / 2);
  p.interleaved = a->interleaved != 0;
  p.amp = static_cast<float>(a->amplitude);
  // the backward kernel turns the gradient back, the forward one with the flag
  p.sign = (kMode == kNormBwd) != (a->inverse != 0) ? -1.f : 1.f;
  p.eps = static_cast<float>(a->eps);
  p.w_f32 = a->weight_dtype == VLAK_F32;
  cudaError_t e = a->dtype == VLAK_F32   ? launch<float, kMode>(p, l.vec, l.blocks, a->n_tensors, cs)
                  : a->dtype == VLAK_F16 ? launch<__half, kMode>(p, l.vec, l.blocks, a->n_tensors, cs)
                                         : launch<__nv_bfloat16, kMode>(p, l.vec, l.blocks, a->n_tensors, cs);
  if (e != cudaSuccess) return set_cuda_error(op, e);
  if (kMode == kNormBwd) {
    DwParams d{};
    for (int i = 0; i < a->n_tensors; ++i) {
      d.part[i] = p.t[i].dw_part;
      d.dw[i] = a->t[i].grad_weight;
      d.rows[i] = l.blocks;
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
