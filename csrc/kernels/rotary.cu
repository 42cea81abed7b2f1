// Rotary positions of queries and keys, alone and with their RMS norm per head, forward and backward.
//
// A pair (a, b) of a head at position t turns by the angle t f_i: a' = a cos - b sin, b' = b cos + a sin; the gradient is the same with -sin. Pairs lie half the
// rotary part apart or side by side, what is behind the rotary part stays. With the norm, n = x r with r = (mean x^2 + eps)^(-1/2) over the head, y = R(n w), and
// with g = R^T dy: dx = r (w g - n mean(w g n)), dw = sum of g n over all rows. r is worked out again in the backward pass, from the row that is read anyhow.
//
// An item is the pairs of one thread: kVec values of the first half and the kVec they turn with (or 2 kVec neighbours), two 16-byte accesses where the
// addresses allow. A block takes a few tokens with all their heads: sines and cosines of a token are worked out once, into shared memory, behind the loads of the
// values. Angles are turns, reduced to half a turn before they become fp32, and known to fp32's last bit at any position (turn_of); that costs some ten 64-bit
// instructions a pair and token, which the heads share. Several heads are one row each of the same launch: q, k and, of a packed projection, v, which is copied.
// With the norm a row's items lie in neighbouring lanes, so that its sums are shuffles, and a thread always holds the same columns, so that dw stays in registers;
// blocks then walk over the tokens, and their partial sums are added up in their order by a second launch (two calls give the same bits).
// What bounds it: without the norm HBM, every value is read once and written once: 34 us for fp32 queries and keys [2, 8191, 12, 64], 5.9 TB/s; a packed bf16 [32, 256, 3, 8, 64] takes
// 11.5 us forward and 15.5 backward, 3.7 TB/s over both, as its tiles are over before the next one's loads are on their way. With the norm neither HBM (30..34 % busy) nor the
// instructions (43..46 % of the issue slots) but the latencies in between: registers leave room for two blocks an SM, and a batch of items is loaded, worked on and stored before the next
// is asked for. [2, 4096, 32 + 8, 128] takes 48 us forward and 80 backward, 3.3 TB/s over both (x is read twice). So instructions come two a piece (packed fp32), weights, sines and
// cosines in 16-byte loads, and the backward pass's two sums in one round of shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../include/flodl_b200.h"
#include "common.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;            // of a tile

template <int kBytes> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// kVec values of one access.
template <typename T, int kVec>
union Pack {
  typename RawOf<sizeof(T) * kVec>::type raw;
  T v[kVec];
  __device__ Pack() {}
};
template <typename T, int kVec>
__device__ __forceinline__ void load(Pack<T, kVec>& p, const T* at) { p.raw = *reinterpret_cast<const decltype(p.raw)*>(at); }
template <typename T, int kVec>
__device__ __forceinline__ void store(const Pack<T, kVec>& p, T* at) { *reinterpret_cast<decltype(p.raw)*>(at) = p.raw; }

// The two accesses of item i: where they start in the head, and the first of its pairs. What does not turn is pairs that do not.
struct ItemAt {
  int a, b, pair;
  bool turns;
};
template <int kVec, bool kSide>
__device__ __forceinline__ ItemAt item_at(int i, int rot) {
  ItemAt w;
  w.turns = i * 2 * kVec < rot;
  w.pair = i * kVec;
  w.a = kSide || !w.turns ? i * 2 * kVec : i * kVec;
  w.b = kSide || !w.turns ? w.a + kVec : w.a + rot / 2;
  return w;
}

// The values of an item as pairs (lo[j], hi[j]), and back. kSide: neighbours, pair j is values 2j and 2j + 1 of a and b one after the other.
template <typename T, int kVec, bool kSide>
__device__ __forceinline__ void unpack(const Pack<T, kVec>& a, const Pack<T, kVec>& b, float (&lo)[kVec], float (&hi)[kVec]) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    lo[j] = to_float(!kSide ? a.v[j] : 2 * j < kVec ? a.v[(2 * j) % kVec] : b.v[(2 * j) % kVec]);
    hi[j] = to_float(!kSide ? b.v[j] : 2 * j + 1 < kVec ? a.v[(2 * j + 1) % kVec] : b.v[(2 * j + 1) % kVec]);
  }
}
template <typename T, int kVec, bool kSide>
__device__ __forceinline__ void pack(Pack<T, kVec>& a, Pack<T, kVec>& b, const float (&lo)[kVec], const float (&hi)[kVec]) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    a.v[j] = from_float<T>(!kSide ? lo[j] : j % 2 ? hi[j / 2] : lo[j / 2]);
    b.v[j] = from_float<T>(!kSide ? hi[j] : (kVec + j) % 2 ? hi[(kVec + j) / 2] : lo[(kVec + j) / 2]);
  }
}
// Columns of the values lo[j] and hi[j].
template <int kVec, bool kSide>
__device__ __forceinline__ int lo_at(const ItemAt& w, int j) { return kSide ? w.a + 2 * j : w.a + j; }
template <int kVec, bool kSide>
__device__ __forceinline__ int hi_at(const ItemAt& w, int j) { return kSide ? w.a + 2 * j + 1 : w.b + j; }

// kN fp32 values in a row of shared memory, in the widest loads.
template <int kN>
__device__ __forceinline__ void load_row(const float* at, float (&v)[kN]) {
  if constexpr (kN % 4 == 0) {
#pragma unroll
    for (int j = 0; j < kN; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(at + j);
      v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) v[j] = at[j];
  }
}
// An item's weights, as pairs.
template <int kVec, bool kSide>
__device__ __forceinline__ void load_weights(const float* w, const ItemAt& at, float (&lo)[kVec], float (&hi)[kVec]) {
  float a[kVec], b[kVec];
  load_row(w + at.a, a);
  load_row(w + at.b, b);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    lo[j] = !kSide ? a[j] : 2 * j < kVec ? a[(2 * j) % kVec] : b[(2 * j) % kVec];
    hi[j] = !kSide ? b[j] : 2 * j + 1 < kVec ? a[(2 * j + 1) % kVec] : b[(2 * j + 1) % kVec];
  }
}

// o = a b + c, a b and a s for kN values, two an instruction. None flushes subnormal values, as the build's own arithmetic does: a turn by nothing gives back what came.
__device__ __forceinline__ F2 whole_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 whole_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
template <int kN>
__device__ __forceinline__ void v_fma(float (&o)[kN], const float (&a)[kN], const float (&b)[kN], const float (&c)[kN]) {
  if constexpr (kN == 1) {
    asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(o[0]) : "f"(a[0]), "f"(b[0]), "f"(c[0]));
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) f2_get(whole_fma(f2_make(a[j], a[j + 1]), f2_make(b[j], b[j + 1]), f2_make(c[j], c[j + 1])), o[j], o[j + 1]);
  }
}
template <int kN>
__device__ __forceinline__ void v_mul(float (&o)[kN], const float (&a)[kN], const float (&b)[kN]) {
  if constexpr (kN == 1) {
    asm("mul.rn.f32 %0, %1, %2;" : "=f"(o[0]) : "f"(a[0]), "f"(b[0]));
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) f2_get(whole_mul(f2_make(a[j], a[j + 1]), f2_make(b[j], b[j + 1])), o[j], o[j + 1]);
  }
}
template <int kN>
__device__ __forceinline__ void v_scale(float (&o)[kN], const float (&a)[kN], float s) {
  float b[kN];
#pragma unroll
  for (int j = 0; j < kN; ++j) b[j] = s;
  v_mul(o, a, b);
}
template <int kN>
__device__ __forceinline__ float v_sum(const float (&a)[kN]) {
  float r = a[0];
#pragma unroll
  for (int j = 1; j < kN; ++j) r += a[j];
  return r;
}
// Pairs (lo, hi) turned: lo cos - hi sin, hi cos + lo sin.
template <int kN>
__device__ __forceinline__ void v_turn(float (&lo)[kN], float (&hi)[kN], const float* cos_at, const float* sin_at) {
  float c[kN], s[kN], minus[kN], a[kN], b[kN];
  load_row(cos_at, c);
  load_row(sin_at, s);
#pragma unroll
  for (int j = 0; j < kN; ++j) minus[j] = -s[j];
  v_mul(a, hi, minus);
  v_mul(b, lo, s);
  v_fma(lo, lo, c, a);
  v_fma(hi, hi, c, b);
}
// The sum over a group of neighbouring lanes, a power of two of them.
__device__ __forceinline__ float group_sum(float v, int group) {
  if (group > 1) v += __shfl_xor_sync(0xffffffffu, v, 1);
  if (group > 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
  if (group > 4) v += __shfl_xor_sync(0xffffffffu, v, 4);
  if (group > 8) v += __shfl_xor_sync(0xffffffffu, v, 8);
  if (group > 16) v += __shfl_xor_sync(0xffffffffu, v, 16);
  return v;
}

// Cosine and sine of x f, position times radians. The turns x f / (2 pi) are a product whose every factor and rounding is carried as two numbers, so that what is left of
// them behind the whole turns is exact to 2^-52 for any whole position. sincospif takes its fp32 part; the rest, below 2^-25, turns the result once more, to first order.
__device__ __forceinline__ void turn_of(double x, double f, float& cs, float& sn) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;        // 1 / (2 pi)
  const double c = __dmul_rn(f, kHi), c_lo = fma(f, kHi, -c) + f * kLo;             // turns a position
  const double t = __dmul_rn(x, c), t_lo = fma(x, c, -t) + x * c_lo;
  const double half = 2.0 * ((t - rint(t)) + t_lo);
  const float a = static_cast<float>(half), rest = static_cast<float>(half - a) * 3.14159265f;
  float s0, c0;
  sincospif(a, &s0, &c0);
  cs = fmaf(-rest, s0, c0);
  sn = fmaf(rest, c0, s0);
}

// One item in flight.
template <typename T, int kVec, bool kBoth>
struct Item {
  Pack<T, kVec> xa, xb;
  Pack<T, kBoth ? kVec : 1> da, db;
  T* y;                     // the head's row of the result; null where there is none to do
  short tok, seg;
};

struct Geometry {
  Div by_group, by_heads, by_seq, by_pairs;
  int tokens, tile, group, items, heads;
  int row;                  // of a token's cosines in shared memory, then its sines: the pairs, rounded up to whole 16-byte accesses
  float inv_d;
};

// Items a thread has in flight. With the norm two: its sums and weights take the registers.
constexpr int items_of(bool norm) { return norm ? 2 : 4; }
// Times that a block's threads are filled by a tile: a block's start (weights, the barrier behind the angles) is shared by as many, but nothing of
// the next tile's is in flight meanwhile. With norms, forward and backward of bf16 queries [2, 4096, 32, 128] and keys [2, 4096, 8, 128] took 174, 132, 129 and
// 143 us with 1, 2, 4 and 8, of a packed [4, 1024, 3, 8, 64] 24.4, 26.1, 21.2 and 21.1. Without, a packed [32, 256, 3, 8, 64] took 27.9, 27.2, 32.7 and 32.7, and the
// forward pass of fp32 queries and keys [2, 8191, 12, 64] 34.9, 34.2, 36.8 and 40.6.
constexpr int passes_of(bool norm) { return norm ? 4 : 2; }

template <typename T, int kVec, bool kSide, bool kNorm, bool kBwd>
__global__ void __launch_bounds__(kThreads, kNorm ? 2 : 3) rotary_kernel(const fb_rotary_args p, const Geometry g) {
  extern __shared__ __align__(16) float turn[];              // [tile][2][row] cos and sin, amplitude included; with the norm, both weights behind them
  constexpr bool kSums = kNorm && kBwd;
  constexpr int kItems = items_of(kNorm);
  const int pairs = p.rot / 2;
  float* weights = turn + g.tile * 2 * g.row;        // [2][D rounded up to 4]
  const int w_row = (p.D + 3) / 4 * 4;
  // with the norm a group is a power of two that divides the threads: the item is the thread's own
  const int own = kNorm ? threadIdx.x & (g.group - 1) : 0;
  float acc[kSums ? 4 : 1][kVec];        // dw of queries and of keys: of lo and of hi
  if constexpr (kSums) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) acc[0][j] = acc[1][j] = acc[2][j] = acc[3][j] = 0.f;
  }
  pdl_entry();
  if constexpr (kNorm) {
    for (int e = threadIdx.x; e < 2 * p.D; e += kThreads) {
      const float* w = p.weight[e >= p.D];
      weights[e >= p.D ? w_row + e - p.D : e] = w ? w[e >= p.D ? e - p.D : e] : 1.f;
    }
  }
  const int n_tiles = (g.tokens + g.tile - 1) / g.tile;
  for (int at = blockIdx.x; at < n_tiles; at += gridDim.x) {
    const int tok0 = at * g.tile, n_tok = min(g.tile, g.tokens - tok0), n = n_tok * g.heads * g.group;
    for (int base = 0; base < n; base += kThreads * kItems) {
      Item<T, kVec, kSums> it[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int idx = base + u * kThreads + threadIdx.x, row = g.by_group(idx), i = kNorm ? own : idx - row * g.group;
        it[u].y = nullptr;
        it[u].seg = 2;
        if (idx < n && i < g.items) {
          const int t = g.by_heads(row);
          int h = row - t * g.heads;
          int seg = 0;
          if (h >= p.heads[0]) { h -= p.heads[0]; seg = 1; }
          if (seg == 1 && h >= p.heads[1]) { h -= p.heads[1]; seg = 2; }
          const int b = g.by_seq(tok0 + t), s = tok0 + t - b * p.S;
          const long long *xs = p.x_strides[seg], *ds = p.dy_strides[seg], *ys = p.y_strides[seg];
          const ItemAt w = item_at<kVec, kSide>(i, p.rot);
          if (!kBwd || (kNorm && seg < 2)) {
            const T* x = static_cast<const T*>(p.x[seg]) + b * xs[0] + s * xs[1] + h * xs[2];
            load(it[u].xa, x + w.a);
            load(it[u].xb, x + w.b);
          }
          if constexpr (kBwd) {
            const T* d = static_cast<const T*>(p.dy[seg]) + b * ds[0] + s * ds[1] + h * ds[2];
            if constexpr (kNorm) {
              load(it[u].da, d + w.a);
              load(it[u].db, d + w.b);
            } else {
              load(it[u].xa, d + w.a);
              load(it[u].xb, d + w.b);
            }
          }
          it[u].y = static_cast<T*>(p.y[seg]) + b * ys[0] + s * ys[1] + h * ys[2];
          it[u].tok = static_cast<short>(t);
          it[u].seg = static_cast<short>(seg);
        }
      }
      if (base == 0) {
        if (at != static_cast<int>(blockIdx.x)) __syncthreads();       // the last tile's have been read
        for (int e = threadIdx.x; e < n_tok * pairs; e += kThreads) {
          const int t = g.by_pairs(e), b = g.by_seq(tok0 + t), s = tok0 + t - b * p.S;
          const long long pos = p.positions ? p.positions[b * p.pos_strides[0] + s * p.pos_strides[1]] : s;
          float sn, cs;
          turn_of(static_cast<double>(pos + p.offset), p.freqs[e - t * pairs], cs, sn);
          float* to = turn + t * 2 * g.row + e - t * pairs;
          to[0] = cs * p.amplitude;
          to[g.row] = (kBwd ? -sn : sn) * p.amplitude;
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int idx = base + u * kThreads + threadIdx.x, i = kNorm ? own : idx - g.by_group(idx) * g.group, seg = it[u].seg;
        const ItemAt w = item_at<kVec, kSide>(i, p.rot);
        float lo[kVec], hi[kVec];
        const float* cos_at = turn + it[u].tok * 2 * g.row + w.pair;
        if constexpr (!kNorm) {
          if (!it[u].y) continue;
          if (seg < 2 && w.turns) {
            unpack<T, kVec, kSide>(it[u].xa, it[u].xb, lo, hi);
            v_turn(lo, hi, cos_at, cos_at + g.row);
            pack<T, kVec, kSide>(it[u].xa, it[u].xb, lo, hi);
          }
          store(it[u].xa, it[u].y + w.a);
          store(it[u].xb, it[u].y + w.b);
        } else {
          const bool here = it[u].y != nullptr, normed = here && seg < 2;
          float x_lo[kVec], x_hi[kVec], w_lo[kVec], w_hi[kVec], t_lo[kVec], t_hi[kVec];
          float sq = 0.f;
          if (normed) {
            unpack<T, kVec, kSide>(it[u].xa, it[u].xb, x_lo, x_hi);
            v_mul(t_lo, x_lo, x_lo);
            v_fma(t_lo, x_hi, x_hi, t_lo);
            sq = v_sum(t_lo);
            load_weights<kVec, kSide>(weights + (seg == 1 ? w_row : 0), w, w_lo, w_hi);
          }
          if constexpr (!kBwd) {
            const float r = rsqrtf(group_sum(sq, g.group) * g.inv_d + p.eps);
            if (normed) {
              v_scale(lo, x_lo, r);
              v_scale(hi, x_hi, r);
              v_mul(lo, lo, w_lo);
              v_mul(hi, hi, w_hi);
              if (w.turns) v_turn(lo, hi, cos_at, cos_at + g.row);
            }
          } else {
            // with S = sum of w g x: mean(w g n) n = x r^2 S / D, so both sums are taken at once, before r is known
            float s = 0.f, e_lo[kVec], e_hi[kVec];
            if (normed) {
              unpack<T, kVec, kSide>(it[u].da, it[u].db, e_lo, e_hi);
              if (w.turns) v_turn(e_lo, e_hi, cos_at, cos_at + g.row);
              v_mul(lo, e_lo, w_lo);
              v_mul(hi, e_hi, w_hi);
              v_mul(t_lo, lo, x_lo);
              v_fma(t_lo, hi, x_hi, t_lo);
              s = v_sum(t_lo);
            }
            sq = group_sum(sq, g.group);
            s = group_sum(s, g.group);
            const float r = rsqrtf(sq * g.inv_d + p.eps), k = -(r * s) * (r * g.inv_d);
            if (normed) {
              v_scale(t_lo, x_lo, r);
              v_scale(t_hi, x_hi, r);
              if (seg == 0) {
                v_fma(acc[0], e_lo, t_lo, acc[0]);
                v_fma(acc[1], e_hi, t_hi, acc[1]);
              } else {
                v_fma(acc[2], e_lo, t_lo, acc[2]);
                v_fma(acc[3], e_hi, t_hi, acc[3]);
              }
#pragma unroll
              for (int j = 0; j < kVec; ++j) t_lo[j] = k;
              v_fma(lo, x_lo, t_lo, lo);
              v_fma(hi, x_hi, t_lo, hi);
              v_scale(lo, lo, r);
              v_scale(hi, hi, r);
            }
          }
          if (here) {
            if constexpr (kBwd) {
              if (normed) pack<T, kVec, kSide>(it[u].da, it[u].db, lo, hi);
              store(it[u].da, it[u].y + w.a);
              store(it[u].db, it[u].y + w.b);
            } else {
              if (normed) pack<T, kVec, kSide>(it[u].xa, it[u].xb, lo, hi);
              store(it[u].xa, it[u].y + w.a);
              store(it[u].xb, it[u].y + w.b);
            }
          }
        }
      }
    }
  }
  if constexpr (kSums) {
    // this block's share of dw: over the groups of a warp, then over the warps, in their order
    float* part = turn;        // [warps][2][D]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        for (int o = 16; o >= g.group; o >>= 1) acc[k][j] += __shfl_xor_sync(0xffffffffu, acc[k][j], o);
    if (lane < g.group && own < g.items) {
      const ItemAt w = item_at<kVec, kSide>(own, p.rot);
#pragma unroll
      for (int seg = 0; seg < 2; ++seg)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          float* row = part + (warp * 2 + seg) * p.D;
          row[lo_at<kVec, kSide>(w, j)] = acc[2 * seg][j];
          row[hi_at<kVec, kSide>(w, j)] = acc[2 * seg + 1][j];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * p.D; e += kThreads) {
      float sum = 0.f;
      for (int k = 0; k < kThreads / 32; ++k) sum += part[k * 2 * p.D + e];
      p.partial[static_cast<long long>(blockIdx.x) * 2 * p.D + e] = sum;
    }
  }
}

// (No read-only loads: they may answer from lines that were in L1 before the kernel before this one wrote them.)
// dw[seg][column] = sum over the blocks' partial sums: 32 columns a block, 32 threads to a column.
__global__ void __launch_bounds__(1024) rotary_dw_kernel(const float* partial, float* dwq, float* dwk, const int blocks, const int D) {
  __shared__ float s[32][33];
  pdl_entry();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), first = threadIdx.x >> 5;
  float sum = 0.f;
  if (col < 2 * D)
    for (int b = first; b < blocks; b += 32) sum += partial[static_cast<long long>(b) * 2 * D + col];
  s[first][threadIdx.x & 31] = sum;
  __syncthreads();
  sum = warp_sum(s[threadIdx.x & 31][first]);
  const int mine = blockIdx.x * 32 + first;
  if ((threadIdx.x & 31) == 0 && mine < 2 * D) {
    if (mine < D) {
      if (dwq) dwq[mine] = sum;
    } else if (dwk) {
      dwk[mine - D] = sum;
    }
  }
}

// The widest access that all addresses allow, in values: whole in 16 bytes, in the halves of the rotary part and in what is behind it.
int widest(const fb_rotary_args& a, int size) {
  const auto fits = [&](int v) {
    if ((a.rot / 2) % v || (a.D - a.rot) % (2 * v)) return false;
    const auto ok = [&](const void* p, const long long* st) {
      return reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && st[0] % v == 0 && st[1] % v == 0 && st[2] % v == 0;
    };
    for (int s = 0; s < 3; ++s) {
      if (a.heads[s] == 0) continue;
      if (a.x[s] && !ok(a.x[s], a.x_strides[s])) return false;
      if (a.backward && !ok(a.dy[s], a.dy_strides[s])) return false;
      if (!ok(a.y[s], a.y_strides[s])) return false;
    }
    return true;
  };
  for (int v = 16 / size; v > 1; v /= 2)
    if (fits(v)) return v;
  return 1;
}

template <typename T, int kVec, bool kSide, bool kNorm, bool kBwd>
int launch(const fb_rotary_args& a, const Geometry& g, int grid, size_t smem, cudaStream_t stream) {
  constexpr auto kern = rotary_kernel<T, kVec, kSide, kNorm, kBwd>;
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kThreads), smem, stream, a, g);
  if (e != cudaSuccess) return static_cast<int>(e);
  if constexpr (kNorm && kBwd) {
    if (a.dw[0] || a.dw[1]) launch_pdl(rotary_dw_kernel, dim3((2 * a.D + 31) / 32), dim3(1024), 0, stream, a.partial, a.dw[0], a.dw[1], grid, a.D);
  }
  return static_cast<int>(cudaGetLastError());
}
template <typename T, int kVec>
int pick(const fb_rotary_args& a, const Geometry& g, int grid, size_t smem, cudaStream_t s) {
  const auto by_side = [&](auto side) {
    constexpr bool kSide = decltype(side)::value;
    if (a.norm) return a.backward ? launch<T, kVec, kSide, true, true>(a, g, grid, smem, s) : launch<T, kVec, kSide, true, false>(a, g, grid, smem, s);
    return a.backward ? launch<T, kVec, kSide, false, true>(a, g, grid, smem, s) : launch<T, kVec, kSide, false, false>(a, g, grid, smem, s);
  };
  return a.interleaved ? by_side(std::true_type()) : by_side(std::false_type());
}

int rotary_blocks() { return 2 * sm_count(); }       // of the backward pass with the norm: those that are resident together

}  // namespace
}  // namespace fb

extern "C" int fb_rotary_partial_rows(void) { return fb::rotary_blocks(); }

extern "C" int fb_rotary(const fb_rotary_args* args, void* stream) {
  using namespace fb;
  if (!args) return -3;
  const fb_rotary_args& a = *args;
  const int size = a.dtype == FLODL_FLOAT32 ? 4 : 2;
  if (a.dtype != FLODL_FLOAT32 && a.dtype != FLODL_BFLOAT16 && a.dtype != FLODL_FLOAT16) return -2;
  const long long heads = static_cast<long long>(a.heads[0]) + a.heads[1] + a.heads[2], tokens = static_cast<long long>(a.B) * a.S;
  if (a.B < 0 || a.S < 0 || a.D < 2 || a.D % 2 || a.rot < 0 || a.rot % 2 || a.rot > a.D || a.heads[0] < 1 || a.heads[1] < 0 || a.heads[2] < 0) return -4;
  if (tokens > 0x7fffffffll) return -4;
  if (tokens == 0) return 0;
  const bool reads_x = !a.backward || a.norm;
  for (int s = 0; s < 3; ++s)
    if (a.heads[s] && (!a.y[s] || (reads_x && !a.x[s]) || (a.backward && !a.dy[s]))) return -3;
  if ((a.rot && !a.freqs) || (a.norm && a.backward && !a.partial)) return -3;
  for (int s = 0; s < 3; ++s)
    if (a.heads[s] && (!aligned(a.x[s], size) || !aligned(a.dy[s], size) || !aligned(a.y[s], size))) return -3;
  if (!aligned(a.freqs, 8) || !aligned(a.positions, 8) || !aligned(a.partial, 4)) return -3;
  for (int s = 0; s < 2; ++s)
    if (!aligned(a.weight[s], 4) || !aligned(a.dw[s], 4)) return -3;
  const int v = widest(a, size), items = a.D / (2 * v);
  int group = items;
  if (a.norm) {
    if (items > 32) return -4;
    for (group = 1; group < items;) group *= 2;
  }
  if (heads * group > 0x7fffffffll / kMaxTokens) return -4;
  // A tile: as many tokens as the threads have items for, fewer where that would leave SMs without a block.
  long long tile = kThreads * items_of(a.norm) * passes_of(a.norm) / (heads * group);
  const long long spread = (tokens + 2 * sm_count() - 1) / (2 * sm_count());
  tile = tile < 1 ? 1 : tile > kMaxTokens ? kMaxTokens : tile;
  if (tile > spread) tile = spread;
  const int row = (a.rot / 2 + 3) / 4 * 4;
  if (row > 0 && tile * row * 8 > 32768) tile = 32768 / (row * 8) > 0 ? 32768 / (row * 8) : 1;
  const long long n_tiles = (tokens + tile - 1) / tile;
  const bool sums = a.norm && a.backward;
  const int grid = static_cast<int>(sums && n_tiles > rotary_blocks() ? rotary_blocks() : n_tiles);
  size_t smem = static_cast<size_t>(tile) * row * 8 + (a.norm ? static_cast<size_t>(a.D + 3) / 4 * 32 : 0);
  if (sums && smem < static_cast<size_t>(kThreads / 32) * 2 * a.D * 4) smem = static_cast<size_t>(kThreads / 32) * 2 * a.D * 4;
  if (smem > 48 * 1024) return -4;
  const auto s = static_cast<cudaStream_t>(stream);
  Geometry g;
  g.tokens = static_cast<int>(tokens);
  g.tile = static_cast<int>(tile);
  g.group = group;
  g.items = items;
  g.heads = static_cast<int>(heads);
  g.row = row;
  g.inv_d = 1.f / static_cast<float>(a.D);
  g.by_group = div_by(group);
  g.by_heads = div_by(heads);
  g.by_seq = div_by(a.S);
  g.by_pairs = div_by(a.rot / 2);
  if (a.dtype == FLODL_FLOAT32) {
    if (v == 4) return pick<float, 4>(a, g, grid, smem, s);
    if (v == 2) return pick<float, 2>(a, g, grid, smem, s);
    return pick<float, 1>(a, g, grid, smem, s);
  }
  const auto by_width = [&](auto t) {
    using T = decltype(t);
    if (v == 8) return pick<T, 8>(a, g, grid, smem, s);
    if (v == 4) return pick<T, 4>(a, g, grid, smem, s);
    if (v == 2) return pick<T, 2>(a, g, grid, smem, s);
    return pick<T, 1>(a, g, grid, smem, s);
  };
  return a.dtype == FLODL_BFLOAT16 ? by_width(__nv_bfloat16()) : by_width(__half());
}
