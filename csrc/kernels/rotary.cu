// Rotary positions of queries and keys, alone and with their RMS norm per head, forward and backward.
//
// A pair (a, b) of a head at position t turns by the angle t f_i: a' = a cos - b sin, b' = b cos + a sin; the gradient is the same with -sin. Pairs lie half the
// rotary part apart or side by side, what is behind the rotary part stays. With the norm, n = x r with r = (mean x^2 + eps)^(-1/2) over the head, y = R(n w), and
// with g = R^T dy: dx = r (w g - n mean(w g n)), dw = sum of g n over all rows. r is worked out again in the backward pass, from the row that is read anyhow.
//
// An item is the pairs of one thread: kVec values of the first half and the kVec they turn with (or 2 kVec neighbours), two 16-byte accesses where the
// addresses allow. A block takes a few tokens with all their heads: sines and cosines of a token are worked out once, into shared memory, behind the loads of the
// values. Angles are turns in 64 bits, reduced to half a turn before they become fp32, so any position is as exact as the first; that costs one 64-bit product and one
// rounding a pair and token, which the heads share. Several heads are one row each of the same launch: q, k and, of a packed projection, v, which is copied.
// With the norm a row's items lie in neighbouring lanes, so that its sums are shuffles, and a thread always holds the same columns, so that dw stays in registers;
// blocks then walk over the tokens, and their partial sums are added up in their order by a second launch (two calls give the same bits).
// What bounds it: HBM. Every value is read once and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../include/flodl_b200.h"
#include "common.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;                 // items a thread has in flight
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

// The two accesses of item i: where they start in the head, and the first of its pairs.
struct ItemAt {
  int a, b, pair;
  bool turns;
};
template <int kVec>
__device__ __forceinline__ ItemAt item_at(int i, int rot, bool interleaved) {
  const int turning = rot / (2 * kVec);
  ItemAt w;
  w.turns = i < turning;
  w.pair = i * kVec;
  const bool side = interleaved || !w.turns;        // neighbours
  w.a = side ? i * 2 * kVec : i * kVec;
  w.b = side ? w.a + kVec : w.a + rot / 2;
  return w;
}

// The values of an item as pairs (lo[j], hi[j]), and back.
template <typename T, int kVec>
__device__ __forceinline__ void unpack(const Pack<T, kVec>& a, const Pack<T, kVec>& b, bool side, float (&lo)[kVec], float (&hi)[kVec]) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    // neighbours: pair j is values 2j and 2j + 1 of a and b one after the other
    const float sl = to_float(2 * j < kVec ? a.v[(2 * j) % kVec] : b.v[(2 * j) % kVec]);
    const float sh = to_float(2 * j + 1 < kVec ? a.v[(2 * j + 1) % kVec] : b.v[(2 * j + 1) % kVec]);
    lo[j] = side ? sl : to_float(a.v[j]);
    hi[j] = side ? sh : to_float(b.v[j]);
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void pack(Pack<T, kVec>& a, Pack<T, kVec>& b, bool side, const float (&lo)[kVec], const float (&hi)[kVec]) {
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    a.v[j] = from_float<T>(side ? (j % 2 ? hi[j / 2] : lo[j / 2]) : lo[j]);
    b.v[j] = from_float<T>(side ? ((kVec + j) % 2 ? hi[(kVec + j) / 2] : lo[(kVec + j) / 2]) : hi[j]);
  }
}

// One item in flight.
template <typename T, int kVec, bool kBoth>
struct Item {
  Pack<T, kVec> xa, xb, da, db;
  T* y;                     // the head's row of the result; null where there is none to do
  short tok, seg;
};

template <typename T, int kVec, bool kNorm, bool kBwd>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const fb_rotary_args p, const int tokens, const int tile, const int group, const int items) {
  extern __shared__ float2 turn[];              // [tile][rot / 2] cos and sin, amplitude included
  constexpr bool kSums = kNorm && kBwd;
  const int pairs = p.rot / 2, heads = p.heads[0] + p.heads[1] + p.heads[2];
  float acc[kSums ? 2 : 1][2 * kVec];
  if constexpr (kSums) {
#pragma unroll
    for (int j = 0; j < 2 * kVec; ++j) acc[0][j] = acc[1][j] = 0.f;
  }
  pdl_entry();
  const int n_tiles = (tokens + tile - 1) / tile;
  for (int at = blockIdx.x; at < n_tiles; at += gridDim.x) {
    const int tok0 = at * tile, n_tok = min(tile, tokens - tok0), n = n_tok * heads * group;
    for (int base = 0; base < n; base += kThreads * kItems) {
      Item<T, kVec, kSums> it[kItems];
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int idx = base + u * kThreads + threadIdx.x, row = idx / group, i = idx - row * group;
        it[u].y = nullptr;
        it[u].seg = 2;
        if (idx < n && i < items) {
          const int t = row / heads;
          int h = row - t * heads;
          int seg = 0;
          if (h >= p.heads[0]) { h -= p.heads[0]; seg = 1; }
          if (seg == 1 && h >= p.heads[1]) { h -= p.heads[1]; seg = 2; }
          const int b = (tok0 + t) / p.S, s = tok0 + t - b * p.S;
          const long long *xs = p.x_strides[seg], *ds = p.dy_strides[seg], *ys = p.y_strides[seg];
          const ItemAt w = item_at<kVec>(i, p.rot, p.interleaved != 0);
          if (!kBwd || (kNorm && seg < 2)) {
            const T* x = static_cast<const T*>(p.x[seg]) + b * xs[0] + s * xs[1] + h * xs[2];
            load(it[u].xa, x + w.a);
            load(it[u].xb, x + w.b);
          }
          if constexpr (kBwd) {
            const T* d = static_cast<const T*>(p.dy[seg]) + b * ds[0] + s * ds[1] + h * ds[2];
            load(it[u].da, d + w.a);
            load(it[u].db, d + w.b);
          }
          it[u].y = static_cast<T*>(p.y[seg]) + b * ys[0] + s * ys[1] + h * ys[2];
          it[u].tok = static_cast<short>(t);
          it[u].seg = static_cast<short>(seg);
        }
      }
      if (base == 0) {
        if (at != static_cast<int>(blockIdx.x)) __syncthreads();       // the last tile's have been read
        for (int e = threadIdx.x; e < n_tok * pairs; e += kThreads) {
          const int t = e / pairs, b = (tok0 + t) / p.S, s = tok0 + t - b * p.S;
          const long long pos = p.positions ? p.positions[b * p.pos_strides[0] + s * p.pos_strides[1]] : s;
          const double turns = static_cast<double>(pos + p.offset) * (p.freqs[e - t * pairs] * 0.15915494309189533577);      // 1 / (2 pi)
          float sn, cs;
          sincospif(2.f * static_cast<float>(turns - rint(turns)), &sn, &cs);
          turn[e] = make_float2(cs * p.amplitude, (kBwd ? -sn : sn) * p.amplitude);
        }
        __syncthreads();
      }
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int idx = base + u * kThreads + threadIdx.x, i = idx % group, seg = it[u].seg;
        const ItemAt w = item_at<kVec>(i, p.rot, p.interleaved != 0);
        const bool side = p.interleaved != 0 || !w.turns;
        float lo[kVec], hi[kVec];
        if constexpr (!kNorm) {
          if (!it[u].y) continue;
          Pack<T, kVec>&ra = kBwd ? it[u].da : it[u].xa, &rb = kBwd ? it[u].db : it[u].xb;
          if (seg < 2 && w.turns) {
            unpack(ra, rb, side, lo, hi);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              const float2 c = turn[it[u].tok * pairs + w.pair + j];
              const float a = lo[j];
              lo[j] = a * c.x - hi[j] * c.y;
              hi[j] = hi[j] * c.x + a * c.y;
            }
            pack(ra, rb, side, lo, hi);
          }
          store(ra, it[u].y + w.a);
          store(rb, it[u].y + w.b);
        } else {
          const bool here = it[u].y != nullptr, normed = here && seg < 2;
          float n_lo[kVec], n_hi[kVec], g_lo[kVec], g_hi[kVec], w_lo[kVec], w_hi[kVec];
          float sq = 0.f;
          if (normed) {
            unpack(it[u].xa, it[u].xb, side, n_lo, n_hi);
#pragma unroll
            for (int j = 0; j < kVec; ++j) sq += n_lo[j] * n_lo[j] + n_hi[j] * n_hi[j];
            const float* wt = p.weight[seg];
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              w_lo[j] = wt ? wt[side ? w.a + 2 * j : w.a + j] : 1.f;
              w_hi[j] = wt ? wt[side ? w.a + 2 * j + 1 : w.b + j] : 1.f;
            }
          }
          for (int o = group >> 1; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          const float r = rsqrtf(sq / p.D + p.eps);
          float dot = 0.f;
          if (normed) {
            if constexpr (kBwd) unpack(it[u].da, it[u].db, side, g_lo, g_hi);
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              float2 c = make_float2(1.f, 0.f);
              if (w.turns) c = turn[it[u].tok * pairs + w.pair + j];
              n_lo[j] *= r;
              n_hi[j] *= r;
              if constexpr (!kBwd) {
                const float a = n_lo[j] * w_lo[j], b = n_hi[j] * w_hi[j];
                lo[j] = a * c.x - b * c.y;
                hi[j] = b * c.x + a * c.y;
              } else {
                const float a = g_lo[j] * c.x - g_hi[j] * c.y, b = g_hi[j] * c.x + g_lo[j] * c.y;
                const float da = a * n_lo[j], db = b * n_hi[j];
                if (seg == 0) {
                  acc[0][2 * j] += da;
                  acc[0][2 * j + 1] += db;
                } else {
                  acc[1][2 * j] += da;
                  acc[1][2 * j + 1] += db;
                }
                g_lo[j] = a * w_lo[j];
                g_hi[j] = b * w_hi[j];
                dot += da * w_lo[j] + db * w_hi[j];
              }
            }
          }
          if constexpr (kBwd) {
            for (int o = group >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            dot /= p.D;
            if (normed) {
#pragma unroll
              for (int j = 0; j < kVec; ++j) {
                lo[j] = r * (g_lo[j] - n_lo[j] * dot);
                hi[j] = r * (g_hi[j] - n_hi[j] * dot);
              }
            }
          }
          if (here) {
            Pack<T, kVec>&ra = kBwd ? it[u].da : it[u].xa, &rb = kBwd ? it[u].db : it[u].xb;
            if (normed) pack(ra, rb, side, lo, hi);
            store(ra, it[u].y + w.a);
            store(rb, it[u].y + w.b);
          }
        }
      }
    }
  }
  if constexpr (kSums) {
    // this block's share of dw: over the groups of a warp, then over the warps, in their order
    float* part = reinterpret_cast<float*>(turn);        // [warps][2][D]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = lane % group;
    __syncthreads();
#pragma unroll
    for (int seg = 0; seg < 2; ++seg)
#pragma unroll
      for (int j = 0; j < 2 * kVec; ++j)
        for (int o = 16; o >= group; o >>= 1) acc[seg][j] += __shfl_xor_sync(0xffffffffu, acc[seg][j], o);
    if (lane < group && i < items) {
      const ItemAt w = item_at<kVec>(i, p.rot, p.interleaved != 0);
      const bool side = p.interleaved != 0 || !w.turns;
#pragma unroll
      for (int seg = 0; seg < 2; ++seg)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          float* row = part + (warp * 2 + seg) * p.D;
          row[side ? w.a + 2 * j : w.a + j] = acc[seg][2 * j];
          row[side ? w.a + 2 * j + 1 : w.b + j] = acc[seg][2 * j + 1];
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

template <typename T, int kVec, bool kNorm, bool kBwd>
int launch(const fb_rotary_args& a, int grid, int tokens, int tile, int group, int items, size_t smem, cudaStream_t stream) {
  constexpr auto kern = rotary_kernel<T, kVec, kNorm, kBwd>;
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kThreads), smem, stream, a, tokens, tile, group, items);
  if (e != cudaSuccess) return static_cast<int>(e);
  if constexpr (kNorm && kBwd) {
    if (a.dw[0] || a.dw[1])
      launch_pdl(rotary_dw_kernel, dim3((2 * a.D + 31) / 32), dim3(1024), 0, stream, a.partial, a.dw[0], a.dw[1], grid, a.D);
  }
  return static_cast<int>(cudaGetLastError());
}
template <typename T, int kVec>
int pick(const fb_rotary_args& a, int grid, int tokens, int tile, int group, int items, size_t smem, cudaStream_t s) {
  if (a.norm) return a.backward ? launch<T, kVec, true, true>(a, grid, tokens, tile, group, items, smem, s) : launch<T, kVec, true, false>(a, grid, tokens, tile, group, items, smem, s);
  return a.backward ? launch<T, kVec, false, true>(a, grid, tokens, tile, group, items, smem, s) : launch<T, kVec, false, false>(a, grid, tokens, tile, group, items, smem, s);
}

int rotary_blocks() { return 4 * sm_count(); }       // of the backward pass with the norm: those that are resident together

}  // namespace
}  // namespace fb

extern "C" int fb_rotary_partial_rows(void) { return fb::rotary_blocks(); }

extern "C" int fb_rotary(const fb_rotary_args* args, void* stream) {
  using namespace fb;
  const fb_rotary_args& a = *args;
  const int size = a.dtype == FLODL_FLOAT32 ? 4 : 2;
  if (a.dtype != FLODL_FLOAT32 && a.dtype != FLODL_BFLOAT16 && a.dtype != FLODL_FLOAT16) return -2;
  const long long heads = static_cast<long long>(a.heads[0]) + a.heads[1] + a.heads[2], tokens = static_cast<long long>(a.B) * a.S;
  if (a.B < 0 || a.S < 0 || a.D < 2 || a.D % 2 || a.rot < 0 || a.rot % 2 || a.rot > a.D || a.heads[0] < 1 || a.heads[1] < 0 || a.heads[2] < 0) return -4;
  if (tokens > 0x7fffffffll) return -4;
  if (tokens == 0) return 0;
  const int v = widest(a, size), items = a.D / (2 * v);
  int group = items;
  if (a.norm) {
    if (items > 32) return -4;
    for (group = 1; group < items;) group *= 2;
  }
  if (heads * group > 0x7fffffffll / kMaxTokens) return -4;
  // A tile: as many tokens as the threads have items for, fewer where that would leave SMs without a block.
  long long tile = kThreads * kItems / (heads * group);
  const long long spread = (tokens + 2 * sm_count() - 1) / (2 * sm_count());
  tile = tile < 1 ? 1 : tile > kMaxTokens ? kMaxTokens : tile;
  if (tile > spread) tile = spread;
  if (a.rot > 0 && tile * a.rot * 4 > 32768) tile = 32768 / (a.rot * 4) > 0 ? 32768 / (a.rot * 4) : 1;
  const long long n_tiles = (tokens + tile - 1) / tile;
  const bool sums = a.norm && a.backward;
  const int grid = static_cast<int>(sums && n_tiles > rotary_blocks() ? rotary_blocks() : n_tiles);
  size_t smem = static_cast<size_t>(tile) * a.rot * 4;
  if (sums && smem < static_cast<size_t>(kThreads / 32) * 2 * a.D * 4) smem = static_cast<size_t>(kThreads / 32) * 2 * a.D * 4;
  if (smem > 48 * 1024) return -4;
  const auto s = static_cast<cudaStream_t>(stream);
  const int ntok = static_cast<int>(tokens), nt = static_cast<int>(tile);
  if (a.dtype == FLODL_FLOAT32) {
    if (v == 4) return pick<float, 4>(a, grid, ntok, nt, group, items, smem, s);
    if (v == 2) return pick<float, 2>(a, grid, ntok, nt, group, items, smem, s);
    return pick<float, 1>(a, grid, ntok, nt, group, items, smem, s);
  }
  const auto by_width = [&](auto t) {
    using T = decltype(t);
    if (v == 8) return pick<T, 8>(a, grid, ntok, nt, group, items, smem, s);
    if (v == 4) return pick<T, 4>(a, grid, ntok, nt, group, items, smem, s);
    if (v == 2) return pick<T, 2>(a, grid, ntok, nt, group, items, smem, s);
    return pick<T, 1>(a, grid, ntok, nt, group, items, smem, s);
  };
  return a.dtype == FLODL_BFLOAT16 ? by_width(__nv_bfloat16()) : by_width(__half());
}
