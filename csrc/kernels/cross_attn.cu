// Attention of queries over keys and values of another length (an encoder's states), forward and backward, head dim 64 and 128, on tcgen05.
//
//   o = softmax(scale q k^T + mask) v;   P from the saved row statistics:   dV = P^T dO,   dS = P (dO V^T - D),   D = rowsum(dO o),   dQ = scale dS K,   dK = scale dS^T Q
//
// Rows. The query heads of a key head lie side by side in memory, so a tile's rows are (query, head) pairs of a power of two `pack` of them, head fastest, which one 5-D
// tensor map gives; what is left of the group is heads of their own. One key head's K and V are so read once for all of them, and few queries fill a tile better.
//
// Masks are of keys. A first, small launch lists each batch row's live blocks of 128 keys: those all of whose keys take part, with nothing added, take the short path, the rest
// go by a table of {scale, addend} for each key, and blocks without a key are left out. A key at -inf is absent: its score is replaced whatever it is, and where
// it meets a product as a row of the streamed operand that row is zeroed in shared memory, so infinities and NaN behind a mask reach nothing. An addend beyond
// 2^100 takes the score's place, as it would in 64 bits. Addends are taken relative to the batch row's largest, so that a mask common to a row's keys costs its
// scores no bits.
//
// Work. A unit is a tile of 128 rows that stays with 128 of what streams past it. As many CTAs as fit the GPU take whole tiles as long as there is one for each of them, side by
// side, so that they stream the same heads out of L2 (with one stretch of all units for each CTA, as long heads of 128 took 287 us against 241). What is left, less
// than a tile each, is cut into equal stretches of units: no last wave, and few queries over many keys fill the GPU as well. A tile that a stretch's border cuts leaves
// fp32 sums behind, which a small second launch adds up in the order of the stretches (two calls give the same bits). Where the forward pass has few tiles, the CTAs of a
// cluster share each of them instead and meet in distributed shared memory, which saves that launch. Tokens, and whatever else is little work, take a forward kernel of their own
// in tiles of sixteen rows.
//
// What bounds it. Tokens: HBM (5.4 TB/s at 268 MB of keys and values). Forward, heads of 128: the tensor cores' 100 cycles for a step of 16 with both operands in shared memory, and the
// softmax warps between them (250 us, 1.1 PFLOP/s at 2 x 16 heads x 2048 x 8192). Heads of 64: the softmax warps' chain of loads from TMEM, maximum, exponentials and store, two
// CTAs an SM (165 us, 0.63 PFLOP/s at 8 x 12 x 1024 x 4096; without its exponentials it would take 121). Backward: seven products in place of five, as keys and rows are
// worked out apart, so that no sum is added up by atomics (2 x 16 x 2048 x 8192 of 128: 0.80 ms, 0.86 PFLOP/s of the five; 0.91 ms where calls follow each other for seconds, at 1.66 GHz under the
// power cap).
//
// Statistics, sums and products are fp32. What is rounded to bf16, once each, and why: P and dS, as operands of the tensor cores, which take fp32 only as tf32, at half the rate and twice the
// shared memory; the results, as their type is; and so the o in D = rowsum(dO o), which the backward pass reads as it was given out, and keeps no second copy of 32 bits. P's rounding is half a
// step, 2^-8 of a probability at most, and the sum that divides is of the P that were not rounded: results are within 0.0021..0.0024 of 64 bits where a rounding of the results alone leaves 0.0017
// (root of the mean square, relative).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../include/flodl_b200.h"
#include "flash_attn_common.cuh"

namespace fb {
namespace {

constexpr int kKeys = 128;                  // keys of a block
constexpr float kHuge = 1.2676506e30f;      // 2^100
constexpr int kWith = 512;                  // more than there are CTAs of a kernel that share a tile
constexpr float kLowest = -3.402823466e38f;

// A row's maximum is -inf where it has no key, and at least kLowest (`seen`) where it has any, so that the two stay apart when parts are joined. No key: zeros, and a
// statistic of +inf, which makes every probability 2^-inf = 0. Keys whose scores are all -inf: a sum of zero, 0 / 0, NaN, as their softmax is, and a statistic of -inf, which
// makes the backward pass's probabilities 2^(-inf + inf).
__device__ __forceinline__ float seen(float top) { return fmaxf(top, kLowest); }
__device__ __forceinline__ float inverse_of(float top, float sum) { return top == -INFINITY ? 0.f : 1.f / sum; }
__device__ __forceinline__ float statistic_of(float top, float sum) { return top == -INFINITY ? INFINITY : top + log2f(sum); }

struct CrossParams {
  int B, Hq, Hk, R, Sk;             // Hq = H / pack rows of heads; R = Sq * pack rows each
  int pack_log2, per_kv;            // log2 of pack; rows of heads that share a key head
  int row_tiles, key_blocks;        // of a row of heads; of a key head
  Div by_row_tiles, by_per_kv, by_key_blocks;
  const void* mask;                 // [B, Sk]: one byte a key (0: absent), or fp32 addends; null: none
  long long mask_stride;
  int mask_bool;
  float scale;
  int table;                        // 1: every block by the table (the short path wants a positive scale)
  // what the mask comes to (null without one): live blocks of a batch row, its largest addend, and [B, key_blocks] of block << 1 | goes by the table, those without a key last
  int* live_count;
  float* base;
  int* live;
  int* before;                      // [2][B + 1] live blocks, and batch rows with any, ahead of a batch row; null for up to kScanned of them
  int* status;
};
constexpr int kScanned = 64;

// 5-D tensor map over [B, S, H, D] bf16 as (D, pack, S, H / pack, B), one 64-wide panel of 128 rows a box.
int make_tmap_rows(CUtensorMap* out, const void* base, int D, int pack, long long S, long long Hq, long long B, long long sb, long long ss, long long sh) {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) != cudaSuccess || qres != cudaDriverEntryPointSuccess) return -1;
    fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  ensure_thread_context();
  // the stride of a dimension of one is never used, but has to be a legal one
  const auto legal = [&](long long stride, long long n) { return static_cast<cuuint64_t>(n > 1 ? stride * 2 : 2 * D); };
  cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(pack), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(B)};
  cuuint64_t strides[4] = {legal(sh, pack), legal(ss, S), legal(sh * pack, Hq), legal(sb, B)};
  cuuint32_t box[5] = {64, static_cast<cuuint32_t>(pack), static_cast<cuuint32_t>(128 / pack), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(r);
}

__device__ __forceinline__ void tma_load_5d(uint32_t smem_dst, const void* tmap, uint64_t* bar, int c0, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      :
      : "r"(smem_dst), "l"(tmap), "r"(smem_u32(bar)), "r"(c0), "r"(0), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// A tile of `rows` rows from row `row0` on, its 64-wide panels one after the other.
template <int kD>
__device__ __forceinline__ void load_tile(uint32_t dst, const void* tmap, uint64_t* bar, int rows, int seq0, int h, int b) {
#pragma unroll
  for (int c = 0; c < kD / 64; ++c) tma_load_5d(dst + c * rows * 128, tmap, bar, c * 64, seq0, h, b);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The addend of a key in units of log2, held at the largest finite values; -inf: the key is absent.
__device__ __forceinline__ float key_addend(const CrossParams& p, int b, int kv) {
  if (kv >= p.Sk) return -INFINITY;
  if (!p.mask) return 0.f;
  const long long at = b * p.mask_stride + kv;
  if (p.mask_bool) return static_cast<const uint8_t*>(p.mask)[at] ? 0.f : -INFINITY;
  const float a = static_cast<const float*>(p.mask)[at];
  return isinf(a) || isnan(a) ? a : fminf(fmaxf(a * kLog2e, -3.402823466e38f), 3.402823466e38f);
}
// What the mask says of a key: {scale, addend beyond `base`}. An addend beyond 2^100 leaves nothing of the score.
__device__ __forceinline__ float2 key_entry(const CrossParams& p, int b, int kv, float base) {
  const float a = key_addend(p, b, kv);
  return make_float2(fabsf(a) < kHuge ? p.scale * kLog2e : 0.f, a - base);
}
// Of a block of 128 keys, by a whole warp: 0 nothing takes part, 1 by the table, 2 all of it with nothing added.
__device__ __forceinline__ int block_state(const CrossParams& p, int b, int blk, int lane) {
  bool any = false, all = true;
#pragma unroll
  for (int i = 0; i < kKeys / 32; ++i) {
    const float a = key_addend(p, b, blk * kKeys + i * 32 + lane);
    any |= a != -INFINITY;
    all &= a == 0.f;
  }
  any = __any_sync(0xffffffffu, any);
  all = __all_sync(0xffffffffu, all);
  return !any ? 0 : all && !p.table ? 2 : 1;
}

// What an earlier kernel of the stream wrote is read past L1, and never with read-only loads (ld.global.nc), which may answer from a line that was there before.
__device__ __forceinline__ int live_of(const CrossParams& p, int b) {
  if (!p.live_count) return p.key_blocks;
  const int n = __ldcg(p.live_count + b);
  return FB_INDEX_OK(n, p.key_blocks + 1ll, 301) ? n : 0;
}
// Entry i of a batch row's list; in place of one that is no block, a block behind the last key.
__device__ __forceinline__ int listed(const CrossParams& p, int b, int i) {
  const int v = __ldcg(p.live + static_cast<long long>(b) * p.key_blocks + i);
  return FB_INDEX_OK(v >> 1, p.key_blocks, 302) ? v : p.key_blocks << 1 | 1;
}
// Live block i of a batch row: {block, whether it goes by the table}.
__device__ __forceinline__ int2 live_block(const CrossParams& p, int b, int i) {
  if (p.live) {
    const int v = listed(p, b, i);
    return make_int2(v >> 1, v & 1);
  }
  return make_int2(i, p.table || (i + 1) * kKeys > p.Sk);
}

// Waits, whatever the block's state, until the copies counted by `bar` have landed: shared memory may not be left while one is on its way to it.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  for (uint32_t it = 0; it < (1u << 20) && !mbar_test(bar, parity); ++it) __nanosleep(20);
}

// A whole warp's wait. Most find the phase already over, and a plain test says so in a quarter of the time (26 cycles against 98 of the waiting loop).
// The loop is one function: inlined at every wait it would more than double the code that a CTA fetches.
__device__ __noinline__ bool warp_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return warp_wait(bar, parity, abort_flag, status, code);
}
__device__ __forceinline__ bool warp_ready(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  return warp_wait_long(bar, parity, abort_flag, status, code);
}

// The loop in place, for waits with registers full: a call would have them moved out of its way (8 x 12 x 1024 x 4096 of 128 columns 214 us against 207).
__device__ __forceinline__ bool warp_ready_here(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  return warp_wait(bar, parity, abort_flag, status, code);
}
// One arrival for a warp whose lanes are all done, by a predicate in place of a branch.
__device__ __forceinline__ void arrive_together(uint64_t* bar, int lane) {
  __syncwarp();
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.eq.s32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
      "}\n" ::"r"(smem_u32(bar)),
      "r"(lane)
      : "memory");
}

// A place in a ring of kN stages, and the parity of its turn.
template <int kN>
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ void next() {
    if (++stage == kN) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// ---- who does what. Tiles go batch row by batch row.
struct Place {
  int b, tile, i;
};
struct Run {
  int b, tile, i0, i1, n;        // a tile's units [i0, i1) of n
};
// kKeyTiles: a tile is a live block of a key head, and the rows of its rows of heads stream past it; otherwise it is 128 rows of a row of heads, and live blocks do.
template <bool kKeyTiles>
__device__ __forceinline__ int tiles_of(const CrossParams& p, int live) { return kKeyTiles ? p.Hk * live : live ? p.Hq * p.row_tiles : 0; }
template <bool kKeyTiles>
__device__ __forceinline__ int length_of(const CrossParams& p, int live) { return kKeyTiles ? p.per_kv * p.row_tiles : live; }

// A CTA's share: tiles c, c + CTAs, ... , `waves` of them, then the stretch [begin, end) of the tiles left.
struct Share {
  int waves;
  Place begin, end;
};
// The CTAs of one kind. Without a mask the numbers here say each one's share; with one, the batch rows' live blocks do.
struct Crew {
  int ctas, whole;               // whole: stretches begin and end with tiles
  int waves, first, each, more;  // the first tile of the stretches; their units, and how many of them have one more
  Div by_ctas, by_length, by_tiles;      // (of a tile, and of a batch row, without a mask)
};
// The batch row into which u falls, and what of u is left there, where a batch row of n live blocks holds `each` a live block or, `by_rows`, `each` if it has any. By a whole warp; {B, 0}
// past the last. Few batch rows are looked through 32 at a time, more (kMany) by a search in 32 parts: 8000 x 2 heads x 17 x 33 with a mask took 3.0 ms forward and 12 backward with the
// look. A kernel has one or the other: with both 32 x 8 heads x 256 x 509 both ways took 121.5 us against 119, as a CTA fetches more code at its start.
struct InRow {
  int b, live, left;
};
template <bool kMany>
__device__ __forceinline__ InRow row_of(const CrossParams& p, unsigned long long u, int lane, unsigned each, bool by_rows) {
  if constexpr (kMany) {
    const int* before = p.before + (by_rows ? p.B + 1 : 0);
    const long long q = static_cast<long long>(u / each);
    int b = 0, n = p.B + 1, ahead = 0;        // before[b] <= q, and the last such is in [b, b + n)
    while (n > 1) {
      const int step = (n + 31) / 32, at = lane * step, v = at < n ? __ldcg(before + b + at) : 0;
      const int k = __popc(__ballot_sync(0xffffffffu, at < n && v <= q)) - 1;
      ahead = __shfl_sync(0xffffffffu, v, k);
      b += k * step;
      n = min(step, n - k * step);
    }
    if (b == p.B) return {p.B, 0, 0};
    const int live = live_of(p, b), left = static_cast<int>(u - static_cast<unsigned long long>(ahead) * each);
    return {b, live, FB_INDEX_OK(left, static_cast<long long>(each) * (by_rows ? 1 : live), 303) ? left : 0};
  }
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int n = b0 + lane < p.B ? live_of(p, b0 + lane) : 0;
    const unsigned long long mine = static_cast<unsigned long long>(by_rows ? n > 0 : n) * each;
    unsigned long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, u < upto);
    if (past) {
      const int k = __ffs(past) - 1;
      return {b0 + k, __shfl_sync(0xffffffffu, n, k), static_cast<int>(u - __shfl_sync(0xffffffffu, upto - mine, k))};
    }
    u -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return {p.B, 0, 0};
}
// The next batch row with a key, B past the last. By a whole warp.
template <bool kMany>
__device__ __forceinline__ int next_row(const CrossParams& p, int b, int lane) {
  if constexpr (kMany) return row_of<true>(p, __ldcg(p.before + p.B + 1 + b) + 1u, lane, 1, true).b;
  do ++b;
  while (b < p.B && live_of(p, b) == 0);
  return b;
}
// Tiles of a batch row: so many a live block (kKeyTiles), or so many if it has any.
template <bool kKeyTiles, bool kMany>
__device__ __forceinline__ InRow row_of_tile(const CrossParams& p, int tile, int lane) {
  return row_of<kMany>(p, static_cast<unsigned>(tile), lane, static_cast<unsigned>(kKeyTiles ? p.Hk : p.Hq * p.row_tiles), !kKeyTiles);
}
template <bool kKeyTiles, bool kMany>
__device__ __forceinline__ Share share_of(const CrossParams& p, const Crew& crew, int cta, int lane) {
  Share s;
  if (!p.live_count) {
    s.waves = crew.waves;
    const int len = length_of<kKeyTiles>(p, p.key_blocks), per_b = tiles_of<kKeyTiles>(p, p.key_blocks);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const int u = crew.each * (cta + k) + min(cta + k, crew.more);
      int tile = crew.by_length(u), i = u - tile * len;
      if (crew.whole && i > 0) {
        ++tile;
        i = 0;
      }
      tile += crew.first;
      const int b = crew.by_tiles(tile);
      (k ? s.end : s.begin) = {b, tile - b * per_b, i};
    }
    return s;
  }
  const unsigned heads = static_cast<unsigned>(p.Hq) * p.row_tiles;        // units of a live block
  const auto live_ahead = [&](int end) {
    if constexpr (kMany) return __ldcg(p.before + end);
    int n = 0;
    for (int b = lane; b < end; b += 32) n += live_of(p, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    return n;
  };
  const int live = live_ahead(p.B);
  int total = live * p.Hk;
  if (!kKeyTiles) {
    int rows = 0;
    if constexpr (kMany) {
      rows = __ldcg(p.before + 2 * p.B + 1);
    } else {
      for (int b0 = 0; b0 < p.B; b0 += 32) rows += __popc(__ballot_sync(0xffffffffu, b0 + lane < p.B && live_of(p, b0 + lane) > 0));
    }
    total = rows * p.Hq * p.row_tiles;
  }
  s.waves = crew.by_ctas(total);
  const int first = s.waves * crew.ctas;
  const unsigned long long all = static_cast<unsigned long long>(live) * heads;
  unsigned long long from = 0;        // units ahead of the first tile of the stretches
  if (first > 0) {
    from = all;
    const InRow at = row_of_tile<kKeyTiles, kMany>(p, first, lane);
    if (at.b < p.B) from = static_cast<unsigned long long>(live_ahead(at.b)) * heads + static_cast<unsigned long long>(at.left) * length_of<kKeyTiles>(p, at.live);
  }
  const int rest = static_cast<int>(all - from), each = crew.by_ctas(rest), more = rest - each * crew.ctas;        // (less than a tile for each CTA)
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const InRow in = row_of<kMany>(p, from + static_cast<unsigned>(each * (cta + k) + min(cta + k, more)), lane, heads, false);
    Place at = {in.b, 0, 0};
    if (at.b < p.B) {
      const int len = length_of<kKeyTiles>(p, in.live);
      at.tile = static_cast<unsigned>(in.left) / static_cast<unsigned>(len);
      at.i = in.left - at.tile * len;
      if (crew.whole && at.i > 0) {
        at.i = 0;
        if (++at.tile == tiles_of<kKeyTiles>(p, in.live)) {
          at.tile = 0;
          at.b = next_row<kMany>(p, at.b, lane);
        }
      }
    }
    (k ? s.end : s.begin) = at;
  }
  return s;
}
// The runs of a share, one after the other, by a whole warp.
template <bool kKeyTiles, bool kMany>
struct Walk {
  Place at, end;
  int waves, tile, step;
  __device__ Walk(const Share& s, int first, int ctas) : at(s.begin), end(s.end), waves(s.waves), tile(first), step(ctas) {}
  __device__ bool next(const CrossParams& p, const Crew& crew, Run& r, int lane) {
    if (waves > 0) {
      InRow in;
      if (!p.live_count) {
        in.b = crew.by_tiles(tile);
        in.live = p.key_blocks;
        in.left = tile - in.b * tiles_of<kKeyTiles>(p, p.key_blocks);
      } else {
        in = row_of_tile<kKeyTiles, kMany>(p, tile, lane);
      }
      const int n = length_of<kKeyTiles>(p, in.live);
      r = {in.b, in.left, 0, n, n};
      tile += step;
      --waves;
      return true;
    }
    if (at.b > end.b || (at.b == end.b && (at.tile > end.tile || (at.tile == end.tile && at.i >= end.i)))) return false;
    const int live = live_of(p, at.b), n = length_of<kKeyTiles>(p, live);
    r = {at.b, at.tile, at.i, at.b == end.b && at.tile == end.tile ? end.i : n, n};
    at.i = 0;
    if (++at.tile == tiles_of<kKeyTiles>(p, live)) {
      at.tile = 0;
      at.b = next_row<kMany>(p, at.b, lane);
    }
    return true;
  }
};

// One block a batch row: its live blocks in their order, then the others, and its largest addend.
__global__ void __launch_bounds__(256) cross_live_kernel(const CrossParams p) {
  __shared__ int state[256], warp_live[8];
  __shared__ float largest[8];
  pdl_entry();
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* live = p.live + static_cast<long long>(b) * p.key_blocks;
  int n_live = 0, n_dead = 0;
  for (int first = 0; first < p.key_blocks; first += 256) {
    const int n = min(256, p.key_blocks - first);
#pragma unroll 4
    for (int j = warp; j < n; j += 8) {
      const int s = block_state(p, b, first + j, lane);
      if (lane == 0) state[j] = s;
    }
    __syncthreads();
    const int s = static_cast<int>(threadIdx.x) < n ? state[threadIdx.x] : 0;
    const unsigned bits = __ballot_sync(0xffffffffu, s != 0);
    if (lane == 0) warp_live[warp] = __popc(bits);
    __syncthreads();
    int before = __popc(bits & ((1u << lane) - 1)), total = 0;
    for (int k = 0; k < 8; ++k) {
      if (k < warp) before += warp_live[k];
      total += warp_live[k];
    }
    if (static_cast<int>(threadIdx.x) < n) {
      const int at = s ? n_live + before : p.key_blocks - 1 - (n_dead + static_cast<int>(threadIdx.x) - before);
      live[at] = (first + static_cast<int>(threadIdx.x)) << 1 | (s == 1);
    }
    n_live += total;
    n_dead += n - total;
    __syncthreads();
  }
  float a = -INFINITY;
  if (!p.mask_bool)
    for (int kv = threadIdx.x; kv < p.Sk; kv += 256) a = fmaxf(a, key_addend(p, b, kv));
  a = warp_max(a);
  if (lane == 0) largest[warp] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 8; ++k) a = fmaxf(a, largest[k]);
    p.base[b] = isinf(a) ? 0.f : a;
    p.live_count[b] = n_live;
  }
}

// One block: `before`, for many batch rows.
__global__ void __launch_bounds__(1024) cross_before_kernel(const CrossParams p) {
  __shared__ int2 of_warp[32];
  pdl_entry();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int2 sum = make_int2(0, 0);        // ahead of this turn's batch rows
  for (int b0 = 0; b0 <= p.B; b0 += 1024) {
    const int b = b0 + static_cast<int>(threadIdx.x), n = b < p.B ? live_of(p, b) : 0;
    int2 upto = make_int2(n, n > 0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto.x, o), y = __shfl_up_sync(0xffffffffu, upto.y, o);
      if (lane >= o) {
        upto.x += x;
        upto.y += y;
      }
    }
    if (lane == 31) of_warp[warp] = upto;
    __syncthreads();
    int2 all = sum;
    for (int k = 0; k < 32; ++k) {
      if (k == warp) sum = all;
      all.x += of_warp[k].x;
      all.y += of_warp[k].y;
    }
    if (b <= p.B) {
      p.before[b] = sum.x + upto.x - n;
      p.before[p.B + 1 + b] = sum.y + upto.y - (n > 0);
    }
    sum = all;
    __syncthreads();        // all have read the warps' sums
  }
}

// What an earlier kernel of the stream wrote is read with plain loads or past L1. A read-only load (ld.global.nc) may answer from a line that was in L1 before the earlier
// kernel wrote it: with programmatic launches that happened about once in 10^4 calls.
// A run as the warp that loads works it out and hands it to the others, two ahead at most: what the others would keep in registers through their loops, or divide for, they
// read from here when they need it.
struct Task {
  int valid, b, h;              // h: of the row of heads, or the key head
  int at;                       // the tile: which 128 rows, or block of keys
  int i0, i1, whole, slot, ends, tile;
  int masked;                   // keys that stay: whether they go by a table
  float base;                   // of the mask
};
template <bool kKeyTiles>
__device__ __forceinline__ Task task_of(const CrossParams& p, const Run& r) {
  int h, per;
  if (!kKeyTiles) {
    per = p.row_tiles;
    h = p.by_row_tiles(r.tile);
  } else if (!p.live_count) {
    per = p.key_blocks;
    h = p.by_key_blocks(r.tile);
  } else {
    per = live_of(p, r.b);
    h = r.tile / per;
  }
  const int tile = r.tile - h * per;
  const int2 at = kKeyTiles ? live_block(p, r.b, tile) : make_int2(tile, 0);
  const bool whole = r.i0 == 0 && r.i1 == r.n;
  return {1, r.b, h, at.x, r.i0, r.i1, whole, r.i0 > 0 ? 0 : 1, r.i1 == r.n, r.tile, at.y, p.base ? __ldcg(p.base + r.b) : 0.f};
}
struct TaskRing {
  uint64_t full[2], empty[2];
  Task task[2];
};
// By the whole loading warp; false after a wait that gave up.
__device__ __forceinline__ bool hand_out(TaskRing& ring, int slot, uint32_t parity, const Task& t, volatile int* abort_flag, int* status, int lane) {
  if (!warp_ready(&ring.empty[slot], parity ^ 1, abort_flag, status, kStatusWaitEmpty)) return false;
  if (lane == 0) ring.task[slot] = t;
  arrive_warp(&ring.full[slot], lane);
  return true;
}

// What a CTA leaves of tiles that its stretch does not hold whole: slot 0 for one that another began, slot 1 for one that it began itself.
struct Left {
  int used, ends, b, tile;       // ends: with this the tile is complete
};

// A thread's row of scores in TMEM, kChunks x 32 columns: each with its key's scale and addend, an absent key's at -inf whatever it was. In place and in a loop: in the
// registers of the common path it would cost that one spills.
template <int kChunks>
__device__ __forceinline__ void apply_table(uint32_t scores, const float2* tb) {
#pragma unroll 1
  for (int c = 0; c < 2 * kChunks; ++c) {
    uint32_t v[16];
    tmem_ld16(scores + 16 * c, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]));
      const float4 k2 = *reinterpret_cast<const float4*>(tb + 16 * c + i);
      v[i] = __float_as_uint(k2.y == -INFINITY ? -INFINITY : fmaf(__uint_as_float(v[i]), k2.x, k2.y));
      v[i + 1] = __float_as_uint(k2.w == -INFINITY ? -INFINITY : fmaf(__uint_as_float(v[i + 1]), k2.z, k2.w));
    }
    tmem_st16(scores + 16 * c, v);
  }
  tmem_st_wait();
}

// Zeroes row `row` of a tile of `rows` rows.
template <int kD>
__device__ __forceinline__ void zero_row(uint32_t tile, int rows, int row) {
#pragma unroll
  for (int c = 0; c < kD / 64; ++c)
#pragma unroll
    for (int g = 0; g < 8; ++g) st_shared_v4(tile + c * rows * 128 + row * 128 + g * 16, make_uint4(0u, 0u, 0u, 0u));
}

// Operands' descriptors. `base` is an offset into the CTA's own memory (in_own): in a cluster an address carries the CTA's number from bit 24 on, which would fall into the
// descriptor's other fields.
__device__ __forceinline__ uint32_t in_own(uint32_t smem) { return smem & 0x3FFFFu; }
__device__ __forceinline__ uint64_t k_desc(uint32_t base, int bytes) { return desc_of(smem_desc_lo(base, 16) + (bytes >> 4), smem_desc_hi(1024)); }
__device__ __forceinline__ uint64_t mn_desc(uint32_t base, int bytes, int lbo) { return desc_of(smem_desc_lo(base, lbo) + (bytes >> 4), smem_desc_hi(1024)); }

__device__ __forceinline__ __nv_bfloat16* out_row(const CrossParams& p, __nv_bfloat16* base, long long sb, long long ss, long long sh, int b, int h, int r) {
  const int g = r & ((1 << p.pack_log2) - 1);
  return base + b * sb + (r >> p.pack_log2) * ss + ((static_cast<long long>(h) << p.pack_log2) + g) * sh;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t smem, int cta) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem), "r"(cta));
  return remote;
}
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_v2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ============================================================================ forward, few rows
// Tiles of sixteen rows, for a token of each sequence and for whatever is as little work. HBM bounds a token, and how long a block of keys takes: a tcgen05 tile has 128 rows
// whatever is in them, and its chain of copy, scores, TMEM, probabilities and product took 1.7 us a block with one warp at work. Here each warp is on its own: it streams
// chunks of keys through a ring of its own with cp.async, one or two in flight, and multiplies them with mma.sync; warps meet at the end, the CTAs that share a tile in
// distributed shared memory or, more than eight of them, by a second launch. Chunks go round all warps of a tile, so that padding at its end takes from each the same.
// Masks are read as the chunks are asked for: absent keys are not copied but filled with zeros, chunks without a key left out.
// One token of 16 x 8 heads of 64 over up to 1500 keys 9.2 us (37 MB; in 128-row tiles 18.4), of 4 x 32 heads of 128 on 4 key heads over 32768 49.9 (5.4 TB/s; 61.3).
template <int kD, int kPerSm>
struct Few {
  static constexpr int kWarps = 4, kStages = kPerSm == 3 ? 2 : 3;        // CTAs on an SM, and the stages that shared memory has room for then
  static constexpr int kChunk = 2048 / kD;                  // keys
  static constexpr int kTile = kChunk * kD * 2;             // bytes of K, and of V
  static constexpr int TAB = 2 * kTile, STAGE = TAB + kChunk * 8, WARP = kStages * STAGE;
  static constexpr int kRow = kD + 8;                       // floats of a row of sums: rows of a quad's warp meet different banks
  static constexpr int SUMS = kWarps * 16 * kRow * 4, ML = SUMS + 16 * kRow * 4, ML_JOINED = ML + kWarps * 16 * 8;
  static constexpr int TOTAL = kWarps * WARP;
  static_assert(ML_JOINED + 16 * 8 <= TOTAL, "sums take the place of the rings");
};
struct FewArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  long long qs[3], ks[3], vs[3], os[3];
  float* stats;                // as in FwdOut
  float* part_o;               // [tiles * parts][16][D] sums relative to the part's maximum; null: the CTAs of a tile are a cluster
  float2* part_ml;             // ... [16] {maximum, sum}
  int parts;                   // CTAs that share a tile
  int row_tiles;               // of sixteen rows
  Div by_parts, by_rows, by_heads;
};
// A tile's place: batch row, row of heads, first row, and how many rows.
struct FewTile {
  int b, h, row0, rows;
};
__device__ __forceinline__ FewTile few_tile(const CrossParams& p, const FewArgs& f, int tile) {
  const int all = f.by_rows(tile), b = f.by_heads(all), row0 = (tile - all * f.row_tiles) * 16;
  return {b, all - b * p.Hq, row0, min(16, p.R - row0)};
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
template <bool kTransposed>
__device__ __forceinline__ void ld_matrices(uint32_t at, uint32_t (&m)[4]) {
  if (kTransposed)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(at) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four columns of a row: the sum of `of` parts' sums, each relative to its own maximum, in their order.
template <typename Ml, typename Sums>
__device__ __forceinline__ void few_join(int of, Ml ml_of, Sums sums_of, float4& acc, float& top, float& sum) {
  top = -INFINITY;
#pragma unroll 4
  for (int k = 0; k < of; ++k) top = fmaxf(top, ml_of(k).x);
  const float ref = top == -INFINITY ? 0.f : top;
  sum = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < of; ++k) {
    const float2 x = ml_of(k);
    const float4 v = sums_of(k);
    const float w = ex2_approx(x.x - ref);
    sum += w * x.y;
    acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
  }
}
__device__ __forceinline__ void few_put(const CrossParams& p, const FewArgs& f, const FewTile& at, int row, int col, float4 acc, float top, float sum) {
  const float inv = inverse_of(top, sum);
  if (f.stats && col == 0) f.stats[(static_cast<long long>(at.b) * p.Hq + at.h) * p.R + at.row0 + row] = statistic_of(top, sum);
  *reinterpret_cast<uint2*>(out_row(p, f.o, f.os[0], f.os[1], f.os[2], at.b, at.h, at.row0 + row) + col * 4) = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
}

template <int kD, int kPerSm>
__global__ void __launch_bounds__(Few<kD, kPerSm>::kWarps * 32, kPerSm) cross_few_kernel(const CrossParams p, const FewArgs f) {
  using L = Few<kD, kPerSm>;
  extern __shared__ __align__(128) uint8_t ring[];
  constexpr int kChunk = L::kChunk, kStages = L::kStages, kCols = kD / 8;        // 16-byte columns of a row
  const int warp = uniform_warp(), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = f.by_parts(blockIdx.x), part = blockIdx.x - tile * f.parts;
  const FewTile at = few_tile(p, f, tile);
  const int b = at.b, h = at.h;
  const uint32_t mine = smem_u32(ring) + warp * L::WARP;
  float2* tab = reinterpret_cast<float2*>(ring + warp * L::WARP + L::TAB);        // of stage 0; others STAGE bytes on
  pdl_entry();

  // rows g and g + 8 of Q, as the products take them
  uint32_t q[kD / 16][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool there = g + r * 8 < at.rows;
    const __nv_bfloat16* row = out_row(p, const_cast<__nv_bfloat16*>(f.q), f.qs[0], f.qs[1], f.qs[2], b, h, at.row0 + (there ? g + r * 8 : 0)) + t * 2;
#pragma unroll
    for (int c = 0; c < kD / 16; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half) q[c][half * 2 + r] = there ? __ldcg(reinterpret_cast<const unsigned*>(row + c * 16 + half * 8)) : 0u;
  }
  const int hk = p.by_per_kv(h), chunks = (p.Sk + kChunk - 1) / kChunk, step = f.parts * L::kWarps;
  const __nv_bfloat16 *k0 = f.k + b * f.ks[0] + hk * f.ks[2], *v0 = f.v + b * f.vs[0] + hk * f.vs[2];
  const float sc = p.scale * kLog2e, base = p.mask && !p.mask_bool ? __ldcg(p.base + b) : 0.f;

  // The mask is read a chunk ahead of the copies, these one or two chunks ahead of the products.
  int c = part * L::kWarps + warp, have = 0;
  unsigned tabled = 0;         // a bit for each stage
  const auto entry_of = [&](int c) {
    const int key = c * kChunk + lane;
    if (lane >= kChunk || key >= p.Sk) return make_float2(sc, -INFINITY);
    return p.mask ? key_entry(p, b, key, base) : make_float2(sc, 0.f);
  };
  float2 ahead = entry_of(c);
  const auto ask = [&]() {
    while (c < chunks) {
      const float2 e = ahead;
      const int first = c * kChunk;
      c += step;
      ahead = entry_of(c);
      const unsigned live = __ballot_sync(0xffffffffu, e.y != -INFINITY);
      if (live == 0) continue;
      const int stage = have % kStages;
      const bool plain = __all_sync(0xffffffffu, lane >= kChunk || (e.x == sc && e.y == 0.f));
      tabled = plain ? tabled & ~(1u << stage) : tabled | 1u << stage;
      if (!plain && lane < kChunk) *reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(tab + lane) + stage * L::STAGE) = e;
#pragma unroll
      for (int j = 0; j < L::kTile / 512; ++j) {
        const int row = (j * 32 + lane) / kCols, col = (j * 32 + lane) % kCols;
        const bool there = live >> row & 1;
        const uint32_t to = mine + stage * L::STAGE + row * (kD * 2) + ((col ^ (row & 7)) << 4);
        const long long key = there ? first + row : 0;
        cp_async16(to, k0 + key * f.ks[1] + col * 8, there);
        cp_async16(to + L::kTile, v0 + key * f.vs[1] + col * 8, there);
      }
      ++have;
      break;
    }
    cp_async_commit();
  };

  float o[kD / 8][4];
#pragma unroll
  for (int n = 0; n < kD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};        // of rows g and g + 8; l of this thread's columns
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) ask();
#pragma unroll 1
  for (int it = 0; it < have; ++it) {
    ask();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const int stage = it % kStages;
    const uint32_t sK = mine + stage * L::STAGE, sV = sK + L::kTile;
    float s[kChunk / 8][4];
#pragma unroll
    for (int n = 0; n < kChunk / 8; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      const int row = n * 8 + (lane & 7);
#pragma unroll
      for (int kk = 0; kk < kD / 32; ++kk) {
        uint32_t w[4];
        ld_matrices<false>(sK + row * (kD * 2) + (((kk * 4 + (lane >> 3)) ^ (lane & 7)) << 4), w);
        mma16(s[n], q[kk * 2], w[0], w[1]);
        mma16(s[n], q[kk * 2 + 1], w[2], w[3]);
      }
    }
    float top[2] = {m[0], m[1]};
    const bool by_table = tabled >> stage & 1;
#pragma unroll
    for (int n = 0; n < kChunk / 8; ++n) {
      float4 e = make_float4(sc, 0.f, sc, 0.f);
      if (by_table) e = *reinterpret_cast<const float4*>(reinterpret_cast<const uint8_t*>(tab + n * 8 + t * 2) + stage * L::STAGE);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        s[n][2 * r] = e.y == -INFINITY ? -INFINITY : fmaf(s[n][2 * r], e.x, e.y);
        s[n][2 * r + 1] = e.w == -INFINITY ? -INFINITY : fmaf(s[n][2 * r + 1], e.z, e.w);
        top[r] = max3(top[r], s[n][2 * r], s[n][2 * r + 1]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      const float a0 = top[0] == -INFINITY ? 1.f : ex2_approx(m[0] - top[0]), a1 = top[1] == -INFINITY ? 1.f : ex2_approx(m[1] - top[1]);
      m[0] = top[0];
      m[1] = top[1];
      l[0] *= a0;
      l[1] *= a1;
#pragma unroll
      for (int n = 0; n < kD / 8; ++n) {
        o[n][0] *= a0;
        o[n][1] *= a0;
        o[n][2] *= a1;
        o[n][3] *= a1;
      }
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < kChunk / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = ex2_approx(s[n][e] - ref[e >> 1]);
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int j = 0; j < kChunk / 16; ++j) {
      const uint32_t a[4] = {pack2(s[2 * j][0], s[2 * j][1]), pack2(s[2 * j][2], s[2 * j][3]), pack2(s[2 * j + 1][0], s[2 * j + 1][1]), pack2(s[2 * j + 1][2], s[2 * j + 1][3])};
      const int row = j * 16 + (lane >> 3 & 1) * 8 + (lane & 7);
#pragma unroll
      for (int n = 0; n < kD / 16; ++n) {
        uint32_t w[4];
        ld_matrices<true>(sV + row * (kD * 2) + (((n * 2 + (lane >> 4)) ^ (lane & 7)) << 4), w);
        mma16(o[2 * n], a, w[0], w[1]);
        mma16(o[2 * n + 1], a, w[2], w[3]);
      }
    }
    __syncwarp();        // the stage may be filled again
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  cp_async_wait<0>();
  __syncthreads();
  // ---- the warps' sums, then the CTAs', in their order
  float* sums = reinterpret_cast<float*>(ring);
  float2* ml = reinterpret_cast<float2*>(ring + L::ML);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = warp * 16 + g + r * 8;
    if (t == 0) ml[row] = make_float2(have ? seen(m[r]) : m[r], l[r]);
#pragma unroll
    for (int n = 0; n < kD / 8; ++n) *reinterpret_cast<float2*>(sums + row * L::kRow + n * 8 + t * 2) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
  }
  __syncthreads();
  float4 acc;
  float top, sum;
  for (int e = threadIdx.x; e < at.rows * (kD / 4); e += L::kWarps * 32) {
    const int row = e / (kD / 4), col = e % (kD / 4);
    few_join(L::kWarps, [&](int k) { return ml[k * 16 + row]; }, [&](int k) { return *reinterpret_cast<const float4*>(sums + (k * 16 + row) * L::kRow + col * 4); }, acc, top, sum);
    if (f.parts == 1) {
      few_put(p, f, at, row, col, acc, top, sum);
    } else if (f.part_o) {
      const long long to = blockIdx.x * 16ll + row;
      *reinterpret_cast<float4*>(f.part_o + to * kD + col * 4) = acc;
      if (col == 0) f.part_ml[to] = make_float2(top, sum);
    } else {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(ring + L::SUMS) + row * L::kRow + col * 4) = acc;
      if (col == 0) *reinterpret_cast<float2*>(ring + L::ML_JOINED + row * 8) = make_float2(top, sum);
    }
  }
  if (f.parts > 1 && !f.part_o) {
    cluster_meet();
    const uint32_t all = smem_u32(ring);
    for (int e = part * (L::kWarps * 32) + threadIdx.x; e < at.rows * (kD / 4); e += f.parts * L::kWarps * 32) {
      const int row = e / (kD / 4), col = e % (kD / 4);
      few_join(f.parts, [&](int k) { return ld_cluster_v2(in_cta(all + L::ML_JOINED + row * 8, k)); },
               [&](int k) { return ld_cluster_v4(in_cta(all + L::SUMS + (row * L::kRow + col * 4) * 4, k)); }, acc, top, sum);
      few_put(p, f, at, row, col, acc, top, sum);
    }
    cluster_meet();        // shared memory is there until all have read it
  }
}
// The parts of a tile that were left in global memory: a block a row, its threads four columns of every so manieth part each, the first of which are on their way before
// their weights are known.
template <int kD>
__global__ void __launch_bounds__(128) cross_few_join_kernel(const CrossParams p, const FewArgs f) {
  constexpr int kLanes = kD / 4, kGroups = 128 / kLanes, kAhead = 4;
  __shared__ float weight[kWith], of_warp[8];
  __shared__ float4 of_group[kGroups][kLanes];
  pdl_entry();
  const int tile = blockIdx.x, row = blockIdx.y;
  const FewTile at = few_tile(p, f, tile);
  if (row >= at.rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = threadIdx.x / kLanes, col = threadIdx.x % kLanes;
  const long long first = static_cast<long long>(tile) * f.parts * 16 + row;
  const auto sums = [&](int k) { return k < f.parts ? __ldcg(reinterpret_cast<const float4*>(f.part_o + (first + k * 16) * kD) + col) : make_float4(0.f, 0.f, 0.f, 0.f); };
  float4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) ahead[i] = sums(group + i * kGroups);
  float2 x[kWith / 128];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWith / 128; ++i) {
    const int k = i * 128 + static_cast<int>(threadIdx.x);
    x[i] = k < f.parts ? __ldcg(f.part_ml + first + k * 16) : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, x[i].x);
  }
  top = warp_max(top);
  if (lane == 0) of_warp[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(of_warp[0], of_warp[1]), fmaxf(of_warp[2], of_warp[3]));
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kWith / 128; ++i) {
    const float w = ex2_approx(x[i].x - ref);
    weight[i * 128 + threadIdx.x] = w;
    sum += w * x[i].y;
  }
  sum = warp_sum(sum);
  if (lane == 0) of_warp[4 + warp] = sum;
  __syncthreads();
  sum = of_warp[4] + of_warp[5] + of_warp[6] + of_warp[7];
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = group; k < f.parts; k += kGroups * kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float4 v = ahead[i];
      const float w = k + i * kGroups < f.parts ? weight[k + i * kGroups] : 0.f;
      acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
      ahead[i] = sums(k + (kAhead + i) * kGroups);
    }
  }
  of_group[group][col] = acc;
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) {
    const float4 v = of_group[k][col];
    acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
  }
  few_put(p, f, at, row, col, acc, top, sum);
}

// ===================================================================================== forward
// Two CTAs an SM, so that one's products run under the other's exponentials. Four softmax warps (a thread is a row and all of a block's keys: with two warps to a row, which
// have to agree on its maximum, 8 x 12 x 1024 x 4096 took 206 us against 176), one that issues products, one that loads. P goes to the second product through TMEM.
constexpr int kFwdThreads = 192;
constexpr float kSlack = 8.f;       // the accumulator is scaled anew once a row's maximum has grown by 2^8: most blocks' maxima grow a little in some row of a warp

__device__ __forceinline__ bool all_of_128(bool mine) {
  uint32_t all;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return all != 0;
}

template <int kD>
struct Fwd {
  static constexpr int kStages = kD == 64 ? 2 : 1;
  static constexpr int kTile = 128 * kD * 2;
  static constexpr int Q = 0;
  static constexpr int K = Q + kTile;
  static constexpr int V = K + kStages * kTile;
  static constexpr int TAB = V + kStages * kTile;        // 2 x 128 x {scale, addend}
  static constexpr int BARS = TAB + 2 * 128 * 8;
  static constexpr int TOTAL = BARS + 512;
  // Columns of TMEM. With 128 values a head P takes the place of the scores that it is made from.
  static constexpr uint32_t S = 0, P = kD == 64 ? 128 : 0, O = kD == 64 ? 192 : 128;
};
struct FwdBars {
  uint64_t q_full, q_empty;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full;             // the scores of a block are in TMEM
  uint64_t s_free;             // ... and in the softmax warps' registers
  uint64_t p_ready;            // the probabilities are in TMEM and O has been rescaled where it had to be
  uint64_t pv_done;            // P V has been added to O: of every block where P has a place of its own, else of a run's last (the next scores tell of the others)
  TaskRing tasks;
  Left left[2];
  uint32_t tmem_slot;
  int abort_flag;
};

struct FwdOut {
  __nv_bfloat16* o;
  long long osb, oss, osh;
  float* stats;                // [B, Hq, R] log2 of the sum of the exponentials, relative to the mask's base; null: not wanted
  Left* left;                  // [CTAs][2]
  float* part_o;               // [CTAs][2][128][D] sums relative to the part's maximum
  float2* part_ml;             // ... [128] {maximum, sum}
  Crew crew;
  int parts;                   // CTAs of a cluster, which share a tile; 0: no clusters
  Div by_parts;
};

// 16-byte chunk c of row t of a tile of fp32 sums in shared memory: a warp's rows, which write the same chunk at a time, meet different banks.
template <int kD>
__device__ __forceinline__ uint32_t shared_chunk(int t, int c) { return (t * (kD / 4) + (c ^ (t & 15))) * 16; }
// The CTAs of a cluster join their parts of a tile, four values a thread, in the order of the parts; each CTA every so manieth group of rows. All threads of all of them,
// whatever became of the waits before.
template <int kD>
__device__ __forceinline__ void join_cluster(const CrossParams& p, const FwdOut& out, const FwdBars& bar, uint32_t sums, uint32_t ml) {
  cluster_meet();
  constexpr int kLanes = kD / 4, kRows = kFwdThreads / kLanes;
  const Task& task = bar.tasks.task[0];
  const int k0 = blockIdx.x - out.by_parts(blockIdx.x) * out.parts, row0 = task.at * 128, rows = min(128, p.R - row0);
  const int c = threadIdx.x % kLanes;
  for (int t = k0 * kRows + threadIdx.x / kLanes; t < rows; t += out.parts * kRows) {
    float m = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < out.parts; ++k) m = fmaxf(m, ld_cluster_v2(in_cta(ml + t * 8, k)).x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < out.parts; ++k) {
      const float2 x = ld_cluster_v2(in_cta(ml + t * 8, k));
      const float4 v = ld_cluster_v4(in_cta(sums + shared_chunk<kD>(t, c), k));
      const float w = ex2_approx(x.x - ref);
      l += w * x.y;
      acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
    }
    const float inv = inverse_of(m, l);
    *reinterpret_cast<uint2*>(out_row(p, out.o, out.osb, out.oss, out.osh, task.b, task.h, row0 + t) + c * 4) = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
    if (out.stats && c == 0) out.stats[(static_cast<long long>(task.b) * p.Hq + task.h) * p.R + row0 + t] = statistic_of(m, l);
  }
  cluster_meet();        // shared memory is there until all have read it
}

template <int kD, bool kMany>
__global__ void __launch_bounds__(kFwdThreads, 2)
cross_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CrossParams p, const FwdOut out) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using L = Fwd<kD>;
  constexpr int kS = L::kStages;
  constexpr bool kOwnP = L::P != L::S;
  static_assert(kOwnP || kS == 1, "waits for V");
  static_assert(sizeof(FwdBars) <= 512, "barriers");
  FwdBars& bar = *reinterpret_cast<FwdBars*>(smem + L::BARS);
  volatile int* abort_flag = &bar.abort_flag;
  float2* tab = reinterpret_cast<float2*>(smem + L::TAB);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, 1);
    mbar_init(&bar.q_empty, 4);
    for (int i = 0; i < 2; ++i) { mbar_init(&bar.k_full[i], 1); mbar_init(&bar.k_empty[i], 1); mbar_init(&bar.v_full[i], 1); mbar_init(&bar.v_empty[i], 1); }
    mbar_init(&bar.s_full, 1);
    mbar_init(&bar.s_free, 4);
    mbar_init(&bar.p_ready, 4);
    mbar_init(&bar.pv_done, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&bar.tasks.full[i], 1); mbar_init(&bar.tasks.empty[i], 5); }
    bar.left[0] = bar.left[1] = Left{0, 0, 0, 0};
    bar.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 4) {
    tmem_alloc<1>(&bar.tmem_slot, 256);
    tmem_relinquish<1>();
  }
  if (warp == 5 && elect_one()) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bar.tmem_slot;
  pdl_entry();       // behind the allocation: the next kernel's may not come before it
  const uint32_t sQ = smem_u32(smem + L::Q), sK = smem_u32(smem + L::K), sV = smem_u32(smem + L::V);

  if (warp == 5) {
    // ------------------------------------------------------------------ loads
    Share share = {};
    if (!out.parts) share = share_of<false, kMany>(p, out.crew, blockIdx.x, lane);
    Walk<false, kMany> walk(share, blockIdx.x, gridDim.x);
    Run r;
    Ring<2> rt;
    Ring<kS> ring;
    int runs = 0, ks = 0, vs = 0;
    bool ok = true;
    while (ok) {
      Task task = {};
      if (out.parts) {
        if (runs == 0) {
          const int tile = out.by_parts(blockIdx.x), k = blockIdx.x - tile * out.parts;
          r.b = out.crew.by_tiles(tile);
          r.tile = tile - r.b * p.Hq * p.row_tiles;
          r.n = live_of(p, r.b);
          r.i0 = out.by_parts(r.n * k);
          r.i1 = out.by_parts(r.n * (k + 1));
          task = task_of<false>(p, r);
          task.whole = 0;
        }
      } else if (walk.next(p, out.crew, r, lane)) {
        task = task_of<false>(p, r);
      }
      ok = hand_out(bar.tasks, rt.stage, rt.parity, task, abort_flag, p.status, lane);
      rt.next();
      if (!ok || !task.valid) break;
      const int hk = p.by_per_kv(task.h);
      ok = warp_ready(&bar.q_empty, (runs & 1) ^ 1, abort_flag, p.status, kStatusWaitEmpty);
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(&bar.q_full, L::kTile);
        load_tile<kD>(sQ, &tmQ, &bar.q_full, 128, (task.at * 128) >> p.pack_log2, task.h, r.b);
      }
      __syncwarp();
      ++runs;
      int2 next = make_int2(0, 0);
      if (r.i0 < r.i1) next = live_block(p, r.b, r.i0);
      for (int i = r.i0; i < r.i1; ++i) {
        const int key0 = next.x * kKeys;
        if (i + 1 < r.i1) next = live_block(p, r.b, i + 1);
        ok = warp_ready(&bar.k_empty[ring.stage], ring.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&bar.k_full[ring.stage], L::kTile);
          load_tile<kD>(sK + ring.stage * L::kTile, &tmK, &bar.k_full[ring.stage], 128, key0, hk, r.b);
        }
        __syncwarp();
        ++ks;
        ok = warp_ready(&bar.v_empty[ring.stage], ring.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(&bar.v_full[ring.stage], L::kTile);
          load_tile<kD>(sV + ring.stage * L::kTile, &tmV, &bar.v_full[ring.stage], 128, key0, hk, r.b);
        }
        __syncwarp();
        ++vs;
        ring.next();
      }
    }
    if (runs > 0) drain(&bar.q_full, (runs - 1) & 1);
    for (int u = max(0, ks - kS); u < ks; ++u) drain(&bar.k_full[u % kS], (u / kS) & 1);
    for (int u = max(0, vs - kS); u < vs; ++u) drain(&bar.v_full[u % kS], (u / kS) & 1);
  } else if (warp == 4) {
    // ------------------------------------------------------------------ products
    const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0), idesc_o = make_idesc_bf16(128, kD, 0, 1);
    Ring<2> rt;
    Ring<kS> rk, rv;
    int it = 0, runs = 0;
    bool ok = true;
    const auto scores = [&]() {
      if (!warp_ready(&bar.k_full[rk.stage], rk.parity, abort_flag, p.status, kStatusWaitFull)) return false;
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          umma_bf16<1>(tmem + L::S, k_desc(in_own(sQ), (k >> 2) * 16384 + (k & 3) * 32), k_desc(in_own(sK) + rk.stage * L::kTile, (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
        umma_commit(&bar.s_full);
        umma_commit(&bar.k_empty[rk.stage]);
      }
      __syncwarp();
      rk.next();
      return true;
    };
    while (ok && warp_ready(&bar.tasks.full[rt.stage], rt.parity, abort_flag, p.status, kStatusWaitFull) && bar.tasks.task[rt.stage].valid) {
      const int n = bar.tasks.task[rt.stage].i1 - bar.tasks.task[rt.stage].i0;
      arrive_warp(&bar.tasks.empty[rt.stage], lane);
      rt.next();
      ok = warp_ready(&bar.q_full, runs & 1, abort_flag, p.status, kStatusWaitFull) && (n == 0 || scores());
      ++runs;
      for (int i = 0; i < n && ok; ++i, ++it) {
        // Where P has a place of its own the next scores may come under this block's exponentials, otherwise right behind the product that reads P: a CTA's products
        // run in the order in which they are issued.
        if (kOwnP && i + 1 < n) {
          ok = warp_ready(&bar.s_free, it & 1, abort_flag, p.status, kStatusWaitEpi) && scores();
          if (!ok) break;
        }
        ok = warp_ready(&bar.p_ready, it & 1, abort_flag, p.status, kStatusWaitEpi) && warp_ready(&bar.v_full[rv.stage], rv.parity, abort_flag, p.status, kStatusWaitFull);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 128 / 16; ++k) umma_bf16_ts(tmem + L::O, tmem + L::P + k * 8, mn_desc(in_own(sV) + rv.stage * L::kTile, k * 2048, 16384), idesc_o, i > 0 || k > 0);
          if (kOwnP || i + 1 == n) umma_commit(&bar.pv_done);
          umma_commit(&bar.v_empty[rv.stage]);
        }
        __syncwarp();
        rv.next();
        if (!kOwnP && i + 1 < n) ok = scores();
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: a thread is a row
    const int t = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const float sc = p.scale * kLog2e;
    Ring<2> rt;
    Ring<kS> rv;
    int it = 0, runs = 0;        // blocks, and runs with any
    bool ok = true;
    // After a wait that gave up the loop over a run's blocks runs out without work, and the four warps go on to the next run or leave together, so that none is missed at
    // the barriers.
    while (all_of_128(warp_ready(&bar.tasks.full[rt.stage], rt.parity, abort_flag, p.status, kStatusWaitFull))) {
      const volatile Task& task = bar.tasks.task[rt.stage];
      if (!task.valid) break;
      const int b = task.b, i0 = task.i0, i1 = task.i1;
      const bool works = warp * 32 < p.R - task.at * 128;        // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f;               // the maximum the accumulator is relative to, and the sum
      const float base = task.base;
      const int ragged = p.table ? i0 : p.Sk / kKeys;        // without a list, the first block that goes by the table
      int next = p.live ? i0 < i1 ? listed(p, b, i0) : 0 : i0 >= ragged;
      for (int i = i0; i < i1; ++i, ++it) {
        const bool tabled = next & 1;
        const float2* tb = tab + (it & 1) * 128;
        if (tabled) {
          const int block = p.live ? next >> 1 : i;
          // A wait for V is one for the turn after the last that is known to be over: with one stage the block before has to have left it, as it has once the scores are there.
          if (kS == 1) ok = ok && warp_ready(&bar.s_full, it & 1, abort_flag, p.status, kStatusWaitAccum);
          const float2 k = key_entry(p, b, block * kKeys + t, base);
          tab[(it & 1) * 128 + t] = k;
          if (p.mask && k.y == -INFINITY && block * kKeys + t < p.Sk && ok) {        // an absent key's values meet a probability of zero (what is behind the last key is zeros)
            ok = mbar_wait(&bar.v_full[rv.stage], rv.parity, abort_flag, p.status, kStatusWaitFull);
            if (ok) zero_row<kD>(sV + rv.stage * L::kTile, 128, t);
          }
          ok = __all_sync(0xffffffffu, ok);
          fence_proxy_async_smem();
          asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        next = !p.live ? i + 1 >= ragged : i + 1 < i1 ? listed(p, b, i + 1) : 0;
        rv.next();
        ok = ok && warp_ready_here(&bar.s_full, it & 1, abort_flag, p.status, kStatusWaitAccum);
        if (!ok) continue;
        tc_fence_after_sync();
        if (!works) {
          if (kOwnP) arrive_warp(&bar.s_free, lane);
          if (kOwnP && i > i0) ok = warp_ready(&bar.pv_done, (it - 1) & 1, abort_flag, p.status, kStatusWaitAccum);
          arrive_warp(&bar.p_ready, lane);
          continue;
        }
        if (tabled) apply_table<4>(tmem + L::S + lanes, tb);        // from here on all blocks are alike
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tmem + L::S + lanes + 32 * c, s[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(s[c][e]));
        if (kOwnP) {
          tc_fence_before_sync();
          arrive_together(&bar.s_free, lane);
        }
        const float mul = tabled ? 1.f : sc, below = tabled ? 0.f : base;        // a key with nothing added is `base` below the largest
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
        const float m_new = fmaxf(m, fmaf(mul, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), -below));
        // Until the product of the block before is over, O is not touched and P not overwritten. Where P takes the place of the scores, these came behind that product.
        bool over = i == i0 || !kOwnP;
        if (i == i0) {
          m = m_new;
        } else {
          // (m is -inf where no key has been seen: its sums are zeros, and stay so whatever they are scaled by)
          if (__any_sync(0xffffffffu, m_new > m + kSlack)) {
            if (!over) {
              ok = warp_ready(&bar.pv_done, (it - 1) & 1, abort_flag, p.status, kStatusWaitAccum);
              if (!ok) continue;
              tc_fence_after_sync();
              over = true;
            }
            const float alpha = m_new == -INFINITY ? 1.f : ex2_approx(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < kD; c += 16) {
              uint32_t v[16];
              tmem_ld16(tmem + L::O + lanes + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * alpha);
              tmem_st16(tmem + L::O + lanes + c, v);
            }
          }
        }
        const F2 mul2 = f2_splat(mul), neg_m = f2_splat(m == -INFINITY ? 0.f : -m - below);
        F2 sum[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float lo, hi;
            f2_get(f2_fma(f2_make(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), mul2, neg_m), lo, hi);
            lo = ex2_approx(lo);
            hi = ex2_approx(hi);
            sum[(e >> 1) & 1] = f2_add(sum[(e >> 1) & 1], f2_make(lo, hi));
            pk[e >> 1] = pack2(lo, hi);
          }
          if (c == 0 && !over) {        // (behind 64, 96 or all 128 exponentials, with P in registers meanwhile, 8 x 12 x 1024 x 4096 took 169, 177 and 180 us, behind 32 of them 168)
            ok = warp_ready_here(&bar.pv_done, (it - 1) & 1, abort_flag, p.status, kStatusWaitAccum);
            tc_fence_after_sync();
          }
          tmem_st16(tmem + L::P + lanes + 16 * c, pk);
        }
        if (!ok) continue;
        float a0, a1;
        f2_get(f2_add(sum[0], sum[1]), a0, a1);
        l += a0 + a1;
        tmem_st_wait();
        tc_fence_before_sync();
        arrive_together(&bar.p_ready, lane);
      }
      // ---- the run's rows
      const bool whole = task.whole;
      const int h = task.h, row0 = task.at * 128, rows = min(128, p.R - row0);
      if (i0 < i1) ok = ok && warp_ready(&bar.pv_done, kOwnP ? (it - 1) & 1 : runs++ & 1, abort_flag, p.status, kStatusWaitAccum);
      if (!whole && t == 0) bar.left[task.slot] = Left{1, task.ends, b, task.tile};
      if (ok && works) {
        tc_fence_after_sync();
        const long long row = (static_cast<long long>(b) * p.Hq + h) * p.R + row0 + t, slot = blockIdx.x * 2ll + task.slot;
        if (i0 < i1) m = seen(m);
        const float inv = whole ? inverse_of(m, l) : 1.f;
        if (out.parts) tab[t] = make_float2(m, l);
        else if (!whole) out.part_ml[slot * 128 + t] = make_float2(m, l);
        else if (out.stats && t < rows) out.stats[row] = statistic_of(m, l);
        float* po = whole ? nullptr : out.part_o + (slot * 128 + t) * kD;
#pragma unroll
        for (int c0 = 0; c0 < kD; c0 += 32) {
          uint32_t v[32];
          if (i0 < i1) {
            tmem_ld32_sync(tmem + L::O + lanes + c0, v);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
          }
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(v[e]) * inv;
          if (out.parts) {       // where K and V were, as `shared_chunk` says
#pragma unroll
            for (int e = 0; e < 32; e += 4) st_shared_v4(sK + shared_chunk<kD>(t, (c0 + e) / 4), make_uint4(__float_as_uint(f[e]), __float_as_uint(f[e + 1]), __float_as_uint(f[e + 2]), __float_as_uint(f[e + 3])));
          } else if (whole) {       // through the warp's 4 KB of each of Q's panels, which every product has read
            stage_half(sQ + (c0 >> 6) * 16384 + warp * 4096, lane, c0 & 32, f);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(po + c0 + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
          }
        }
        if (whole) {
          __syncwarp();
          const int sub = lane >> 3, ch = lane & 7;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int rr = k * 4 + sub;
            if (warp * 32 + rr < rows) {
              __nv_bfloat16* dst = out_row(p, out.o, out.osb, out.oss, out.osh, b, h, row0 + warp * 32 + rr) + ch * 8;
#pragma unroll
              for (int c = 0; c < kD / 64; ++c)
                *reinterpret_cast<uint4*>(dst + c * 64) = ld_shared_v4(sQ + c * 16384 + warp * 4096 + rr * 128 + ((ch ^ (rr & 7)) << 4));
            }
          }
          fence_proxy_async_smem();        // the next Q comes to the same place
        }
        tc_fence_before_sync();
      }
      arrive_warp(&bar.q_empty, lane);
      arrive_warp(&bar.tasks.empty[rt.stage], lane);
      rt.next();
    }
    if (t == 0 && !out.parts && !out.crew.whole) {
      out.left[blockIdx.x * 2] = bar.left[0];
      out.left[blockIdx.x * 2 + 1] = bar.left[1];
    }
    // batch rows without a key: zeros
    if (p.live_count)
      for (int b = blockIdx.x; b < p.B; b += gridDim.x)
        if (live_of(p, b) == 0)
          for (long long e = t; e < static_cast<long long>(p.Hq) * p.R * (kD / 8); e += 128) {
            const int c = static_cast<int>(e % (kD / 8)), row = static_cast<int>(e / (kD / 8) % p.R), h = static_cast<int>(e / (kD / 8) / p.R);
            *reinterpret_cast<uint4*>(out_row(p, out.o, out.osb, out.oss, out.osh, b, h, row) + c * 8) = make_uint4(0u, 0u, 0u, 0u);
            if (out.stats && c == 0) out.stats[(static_cast<long long>(b) * p.Hq + h) * p.R + row] = INFINITY;
          }
  }
  if (out.parts) join_cluster<kD>(p, out, bar, sK, smem_u32(tab));
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, 256);
  }
}

// The CTAs that share the tile which `cta` began and did not end, in their order, into `with`; returns how many. By a whole block; at most kWith.
__device__ __forceinline__ int sharers(const Left* left, int cta, int stop, short* with, int* count) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int n = 1;
    if (lane == 0) with[0] = static_cast<short>(cta);
    for (int k0 = cta + 1; k0 < stop; k0 += 32) {
      const Left l = k0 + lane < stop ? left[(k0 + lane) * 2] : Left{0, 0, 0, 0};        // (a stretch may be empty where blocks are masked)
      const unsigned ends = __ballot_sync(0xffffffffu, l.ends), upto = ends ? (2u << (__ffs(ends) - 1)) - 1 : 0xffffffffu;
      const unsigned used = __ballot_sync(0xffffffffu, l.used) & upto;
      if (used >> lane & 1) with[n + __popc(used & ((1u << lane) - 1))] = static_cast<short>(k0 + lane);
      n += __popc(used);
      if (ends) break;
    }
    if (lane == 0) *count = n;
  }
  __syncthreads();
  return *count;
}

// The stretches' shares of a tile joined, by the block of the CTA that began it: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i, four values a thread.
template <int kD>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossParams p, const FwdOut out, const int ctas) {
  __shared__ short with[kWith];
  __shared__ int count;
  pdl_entry();
  constexpr int kLanes = kD / 4;
  const Left first = out.left[blockIdx.x * 2 + 1];
  if (!first.used || !FB_INDEX_OK(first.b, p.B, 304) || !FB_INDEX_OK(first.tile, static_cast<long long>(p.Hq) * p.row_tiles, 305)) return;
  const int n = sharers(out.left, blockIdx.x, ctas, with, &count);
  const int h = first.tile / p.row_tiles, row0 = (first.tile - h * p.row_tiles) * 128, rows = min(128, p.R - row0);
  const int c = (threadIdx.x % kLanes) * 4, t = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes;
  if (t >= rows) return;
  const auto at = [&](int k) { return (with[k] * 2ll + (k == 0)) * 128 + t; };
  float m = -INFINITY;
#pragma unroll 8
  for (int k = 0; k < n; ++k) m = fmaxf(m, out.part_ml[at(k)].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float2 ml = out.part_ml[at(k)];
    const float4 v = *reinterpret_cast<const float4*>(out.part_o + at(k) * kD + c);
    const float w = ex2_approx(ml.x - ref);
    l += w * ml.y;
    acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
  }
  const float inv = inverse_of(m, l);
  __nv_bfloat16* dst = out_row(p, out.o, out.osb, out.oss, out.osh, first.b, h, row0 + t) + c;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
  if (out.stats && c == 0) out.stats[(static_cast<long long>(first.b) * p.Hq + h) * p.R + row0 + t] = statistic_of(m, l);
}

// ==================================================================================== backward
// Two kinds of CTAs, in one launch, one an SM. Both keep a tile of 128 rows of two tensors in shared memory and stream tiles of 128 rows of the other two:
//   keys:  K, V stay; Q, dO stream.   S^T = K Q^T, dP^T = V dO^T;   dV += P^T dO,  dK += dS^T Q
//   rows:  Q, dO stay; K, V stream.   S = Q K^T,   dP = dO V^T;     dQ += dS K
// Scores are so worked out twice, but P and dS reach their products in TMEM, in the place of the scores and the dP that they are made from, and never through shared memory,
// and every gradient is summed in the order of the tiles, with no atomics. Sixteen softmax
// warps: a thread is a row of the tile that stays and 32 of the streamed tile's columns. (With eight, 64 columns each, a warp's exponentials alone took 1050 cycles where the
// unit needs 512: two warps a scheduler do not hide the latencies.) Products of one CTA run in the order in which they are issued, so that what overwrites a place may be
// issued right behind what reads it: S(j+1) behind dV(j) (ahead of time, where there is a second buffer), dP(j+1) behind dK(j) or dQ(j).
// Tiles of 128 columns, not two of 64: with both operands in shared memory a product of 128 x 64 x 16 takes the 64 cycles of one of 128 x 128 x 16.
constexpr int kBwdSoftmaxWarps = 16;
constexpr int kBwdThreads = 32 * (kBwdSoftmaxWarps + 3);        // ... one that issues products, one that loads, one that fills tables

template <int kD>
struct Bwd {
  // Streamed tiles that are there at a time: of Q or K (A), of dO or V (B). A block of V has done its work with dP; Q, K and dO are read again by the products behind.
  static constexpr int stages_a(bool keys) { return kD == 64 ? 3 : keys ? 2 : 3; }
  static constexpr int stages_b(bool keys) { return kD == 64 ? 3 : keys ? 2 : 1; }
  static constexpr int kTile = 128 * kD * 2;
  static constexpr int F0 = 0, F1 = kTile;
  static constexpr int RING = 2 * kTile;                           // A's tiles, then B's
  static constexpr int TAB = RING + (kD == 64 ? 6 : 4) * kTile;    // 3 x 256 floats
  static constexpr int BARS = TAB + 3 * 1024;
  static constexpr int TOTAL = BARS + 512;
  // Columns of TMEM: one more buffer of scores where the accumulators leave room for it.
  static constexpr uint32_t S = 0, DP = 128, ACC0 = 256, ACC1 = 256 + kD;
  static constexpr uint32_t S2_KEYS = 384, S2_ROWS = kD == 64 ? 384 : 256;
  static constexpr bool kTwoForKeys = kD == 64;
};
static_assert(Bwd<128>::TOTAL + 1024 <= 227 * 1024, "shared memory budget");

struct BwdOut {
  const float* stats;              // of the forward pass
  const float* D;                  // [B, Hq, R]
  __nv_bfloat16 *dq, *dk, *dv;
  long long qsb, qss, qsh, ksb, kss, ksh;
  Left* left;                      // [CTAs][2]
  float* part;                     // [CTAs][2][128][D], of the CTAs of keys twice that: dK, then dV
  int key_ctas;
  Crew keys, rows;
};

// P of 32 columns of a thread's scores, as fp32 in `pr` and, for keys, as bf16 in TMEM: P = 2^(mul s - l), with l of the thread's row or, where the columns are rows, -l of `tb`.
template <bool kKeys>
__device__ __forceinline__ void make_p(uint32_t tS, float mul, const float* tb, float neg_l, uint32_t (&pr)[32]) {
  tmem_ld32_sync(tS, pr);
  const F2 mul2 = f2_splat(mul);
  uint32_t pk[16];
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    F2 nl[2] = {f2_splat(neg_l), f2_splat(neg_l)};
    if (kKeys) {
      const float4 x = *reinterpret_cast<const float4*>(tb + e);
      nl[0] = f2_make(x.x, x.y);
      nl[1] = f2_make(x.z, x.w);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int at = e + 2 * k;
      float lo, hi;
      f2_get(f2_fma(f2_make(__uint_as_float(pr[at]), __uint_as_float(pr[at + 1])), mul2, nl[k]), lo, hi);
      lo = ex2_approx(lo);
      hi = ex2_approx(hi);
      pr[at] = __float_as_uint(lo);
      pr[at + 1] = __float_as_uint(hi);
      if (kKeys) pk[at >> 1] = pack2(lo, hi);
    }
  }
  if (kKeys) tmem_st16(tS, pk);
}
// dS = P (dP - D) of the same columns, as bf16 in TMEM.
template <bool kKeys>
__device__ __forceinline__ void make_ds(uint32_t tDP, const float* tb, float neg_d, const uint32_t (&pr)[32]) {
  uint32_t d[32], dk[16];
  tmem_ld32_sync(tDP, d);
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    F2 nd[2] = {f2_splat(neg_d), f2_splat(neg_d)};
    if (kKeys) {
      const float4 y = *reinterpret_cast<const float4*>(tb + e);
      nd[0] = f2_make(y.x, y.y);
      nd[1] = f2_make(y.z, y.w);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int at = e + 2 * k;
      float lo, hi;
      f2_get(f2_mul(f2_make(__uint_as_float(pr[at]), __uint_as_float(pr[at + 1])), f2_add(f2_make(__uint_as_float(d[at]), __uint_as_float(d[at + 1])), nd[k])), lo, hi);
      dk[at >> 1] = pack2(lo, hi);
    }
  }
  tmem_st16(tDP, dk);
}

struct BwdBars {
  uint64_t f_full, f_empty;           // the tiles that stay
  uint64_t a_full[3], a_empty[3];     // a streamed tile of Q or K has landed; every product that reads it has retired
  uint64_t b_full[3], b_empty[3];     // ... of dO or V
  uint64_t tab_full[3];               // A's table is written
  uint64_t s_full[2], dp_full;        // scores and dP are in TMEM
  uint64_t p_ready[2], ds_ready;      // ... and P (one for each place of scores: a warp may be a turn ahead of another there) and dS in their place
  uint64_t acc_done;                  // every product of a run has retired
  TaskRing tasks;
  Left left[2];
  uint32_t tmem_slot;
  int abort_flag;
};

template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_products(BwdBars& bar, const CrossParams& p, uint32_t tmem, uint32_t smem) {
  using L = Bwd<kD>;
  int* status = p.status;
  volatile int* abort_flag = &bar.abort_flag;
  constexpr bool kTwo = !kKeys || L::kTwoForKeys;
  constexpr int kA = L::stages_a(kKeys), kB = L::stages_b(kKeys);
  const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0), idesc_acc = make_idesc_bf16(128, kD, 0, 1);
  Ring<kA> ra, fa;        // of the scores, and of the products that read the tile again
  Ring<kB> rb, fb;
  int it = 0;
  const auto s_at = [&](int n) { return tmem + (kTwo && (n & 1) ? (kKeys ? L::S2_KEYS : L::S2_ROWS) : L::S); };
  const auto a_at = [&](int stage) { return smem + L::RING + stage * L::kTile; };
  const auto b_at = [&](int stage) { return smem + L::RING + (kA + stage) * L::kTile; };
  const auto scores = [&](int n) {
    if (!warp_ready(&bar.a_full[ra.stage], ra.parity, abort_flag, status, kStatusWaitFull)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kD / 16; ++k)
        umma_bf16<1>(s_at(n), k_desc(smem + L::F0, (k >> 2) * 16384 + (k & 3) * 32), k_desc(a_at(ra.stage), (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
      umma_commit(&bar.s_full[kTwo ? n & 1 : 0]);
    }
    __syncwarp();
    ra.next();
    return true;
  };
  const auto dp = [&](bool last) {
    if (!warp_ready(&bar.b_full[rb.stage], rb.parity, abort_flag, status, kStatusWaitFull)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kD / 16; ++k)
        umma_bf16<1>(tmem + L::DP, k_desc(smem + L::F1, (k >> 2) * 16384 + (k & 3) * 32), k_desc(b_at(rb.stage), (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
      umma_commit(&bar.dp_full);
      if (!kKeys) umma_commit(&bar.b_empty[rb.stage]);
      if (last) umma_commit(&bar.f_empty);
    }
    __syncwarp();
    rb.next();
    return true;
  };
  // acc += (the 128 columns, each 32 left as bf16 in the first half of their place) x (the 128 rows of a streamed tile)
  const auto accumulate = [&](uint32_t acc, uint32_t from, uint32_t tile, bool first, uint64_t* ready, uint32_t parity, uint64_t* empty, bool done) {
    if (!warp_ready(ready, parity, abort_flag, status, kStatusWaitEpi)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < 8; ++k) umma_bf16_ts(tmem + acc, from + (k >> 1) * 32 + (k & 1) * 8, mn_desc(tile, k * 2048, 16384), idesc_acc, !first || k > 0);
      umma_commit(empty);
      if (done) umma_commit(&bar.acc_done);
    }
    __syncwarp();
    return true;
  };
  Ring<2> rt;
  bool ok = true;
  for (int runs = 0; ok && warp_ready(&bar.tasks.full[rt.stage], rt.parity, abort_flag, status, kStatusWaitFull) && bar.tasks.task[rt.stage].valid; ++runs) {
    const int n = bar.tasks.task[rt.stage].i1 - bar.tasks.task[rt.stage].i0;
    arrive_warp(&bar.tasks.empty[rt.stage], static_cast<int>(threadIdx.x & 31));
    rt.next();
    ok = warp_ready(&bar.f_full, runs & 1, abort_flag, status, kStatusWaitFull) && scores(it) && dp(n == 1);
    for (int i = 0; i < n && ok; ++i, ++it) {
      const bool more = i + 1 < n, first = i == 0;
      if (kTwo && more) ok = scores(it + 1);
      if (kKeys) {
        ok = ok && accumulate(L::ACC0, s_at(it), b_at(fb.stage), first, &bar.p_ready[kTwo ? it & 1 : 0], (kTwo ? it >> 1 : it) & 1, &bar.b_empty[fb.stage], false);
        fb.next();
        if (!kTwo && more) ok = ok && scores(it + 1);
      }
      ok = ok && accumulate(L::ACC1, tmem + L::DP, a_at(fa.stage), first, &bar.ds_ready, it & 1, &bar.a_empty[fa.stage], !more);
      fa.next();
      if (more) ok = ok && dp(i + 2 == n);
    }
  }
}

template <int kD, bool kKeys, bool kMany>
__device__ __forceinline__ void bwd_loads(BwdBars& bar, const CrossParams& p, const Crew& crew, int first, uint32_t smem, const void* f0, const void* f1, const void* a, const void* b) {
  using L = Bwd<kD>;
  constexpr int kA = L::stages_a(kKeys), kB = L::stages_b(kKeys);
  volatile int* abort_flag = &bar.abort_flag;
  Ring<kA> ra;
  Ring<kB> rb;
  int as = 0, bs = 0, runs = 0;
  const int lane = threadIdx.x & 31;
  Walk<kKeys, kMany> walk(share_of<kKeys, kMany>(p, crew, first, lane), first, crew.ctas);
  Run r;
  Ring<2> rt;
  bool ok = true;
  while (ok) {
    Task task = {};
    if (walk.next(p, crew, r, lane)) task = task_of<kKeys>(p, r);
    ok = hand_out(bar.tasks, rt.stage, rt.parity, task, abort_flag, p.status, lane);
    rt.next();
    if (!ok || !task.valid) break;
    // keys: the tile is a live block of a key head, whose rows of heads' rows stream; rows: 128 rows of a row of heads, and its key head's blocks stream
    const int h = task.h, at0 = kKeys ? task.at * 128 : (task.at * 128) >> p.pack_log2;
    const int past = kKeys ? p.by_row_tiles(r.i0) : 0;
    int head = kKeys ? h * p.per_kv + past : p.by_per_kv(h), row = kKeys ? r.i0 - past * p.row_tiles : 0;
    ok = warp_ready(&bar.f_empty, (runs & 1) ^ 1, abort_flag, p.status, kStatusWaitEmpty);
    if (!ok) break;
    if (elect_one()) {
      mbar_expect_tx(&bar.f_full, 2 * L::kTile);
      load_tile<kD>(smem + L::F0, f0, &bar.f_full, 128, at0, h, r.b);
      load_tile<kD>(smem + L::F1, f1, &bar.f_full, 128, at0, h, r.b);
    }
    __syncwarp();
    ++runs;
    int2 next = make_int2(0, 0);
    if (!kKeys) next = live_block(p, r.b, r.i0);
    for (int i = r.i0; i < r.i1; ++i) {
      const int seq = kKeys ? (row * 128) >> p.pack_log2 : next.x * 128;
      if (!kKeys && i + 1 < r.i1) next = live_block(p, r.b, i + 1);
      ok = warp_ready(&bar.a_empty[ra.stage], ra.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty);
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(&bar.a_full[ra.stage], L::kTile);
        load_tile<kD>(smem + L::RING + ra.stage * L::kTile, a, &bar.a_full[ra.stage], 128, seq, head, r.b);
      }
      __syncwarp();
      ++as;
      ok = warp_ready(&bar.b_empty[rb.stage], rb.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty);
      if (!ok) break;
      if (elect_one()) {
        mbar_expect_tx(&bar.b_full[rb.stage], L::kTile);
        load_tile<kD>(smem + L::RING + (kA + rb.stage) * L::kTile, b, &bar.b_full[rb.stage], 128, seq, head, r.b);
      }
      __syncwarp();
      ++bs;
      ra.next();
      rb.next();
      if (kKeys && ++row == p.row_tiles) {
        row = 0;
        ++head;
      }
    }
  }
  if (runs > 0) drain(&bar.f_full, (runs - 1) & 1);
  for (int u = max(0, as - kA); u < as; ++u) drain(&bar.a_full[u % kA], (u / kA) & 1);
  for (int u = max(0, bs - kB); u < bs; ++u) drain(&bar.b_full[u % kB], (u / kB) & 1);
}

// The table of a streamed tile: {-l[128], -D[128]} of its rows, or its keys' entries.
template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_tables(BwdBars& bar, const CrossParams& p, float* tab, const float* stats, const float* D, int lane) {
  Ring<Bwd<kD>::stages_a(kKeys)> ra;
  Ring<2> rt;
  while (warp_ready(&bar.tasks.full[rt.stage], rt.parity, &bar.abort_flag, p.status, kStatusWaitFull)) {
    const Task r = bar.tasks.task[rt.stage];
    arrive_warp(&bar.tasks.empty[rt.stage], lane);
    rt.next();
    if (!r.valid) return;
    const float base = r.base, shift = kKeys && !r.masked ? base : 0.f;        // keys with nothing added are `base` below the largest
    const int past = kKeys ? p.by_row_tiles(r.i0) : 0;
    int head = kKeys ? r.h * p.per_kv + past : 0, row = kKeys ? r.i0 - past * p.row_tiles : 0;
    for (int i = r.i0; i < r.i1; ++i) {
      float* tb = tab + ra.stage * 256;
      float2 v[4];
      const int2 blk = kKeys ? make_int2(0, 1) : live_block(p, r.b, i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kKeys) {
          const int n = row * 128 + e * 32 + lane;
          const long long line = (static_cast<long long>(r.b) * p.Hq + head) * p.R + n;
          v[e] = make_float2(-INFINITY, 0.f);
          if (n < p.R) v[e] = make_float2(-__ldcg(stats + line) - shift, -__ldcg(D + line));
        } else if (blk.y) {
          v[e] = key_entry(p, r.b, blk.x * 128 + e * 32 + lane, base);
        }
      }
      if (!warp_ready(&bar.a_empty[ra.stage], ra.parity ^ 1, &bar.abort_flag, p.status, kStatusWaitEmpty)) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = e * 32 + lane;
        if (kKeys) {
          tb[n] = v[e].x;
          tb[128 + n] = v[e].y;
        } else if (blk.y) {
          reinterpret_cast<float2*>(tb)[n] = v[e];
        }
      }
      arrive_warp(&bar.tab_full[ra.stage], lane);
      ra.next();
      if (kKeys && ++row == p.row_tiles) {
        row = 0;
        ++head;
      }
    }
  }
}

// A tile whose keys go by a table: the scores with their keys' scales and addends, as in the forward pass, in place.
template <bool kKeys>
__device__ __noinline__ void masked_scores(uint32_t tS, float2 entry, const float2* tb) {
  if (!kKeys) return apply_table<1>(tS, tb);
#pragma unroll 1
  for (int c = 0; c < 32; c += 16) {
    uint32_t v[16];
    tmem_ld16(tS + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      asm volatile("" : "+r"(v[e]));
      v[e] = __float_as_uint(entry.y == -INFINITY ? -INFINITY : fmaf(__uint_as_float(v[e]), entry.x, entry.y));
    }
    tmem_st16(tS + c, v);
  }
  tmem_st_wait();
}
// ... and nothing is left of an absent key's dP.
template <bool kKeys>
__device__ __noinline__ void masked_dp(uint32_t tDP, float2 entry, const float2* tb) {
#pragma unroll 1
  for (int c = 0; c < 32; c += 16) {
    uint32_t v[16];
    tmem_ld16(tDP + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      asm volatile("" : "+r"(v[e]));
      if ((kKeys ? entry.y : tb[c + e].y) == -INFINITY) v[e] = 0u;
    }
    tmem_st16(tDP + c, v);
  }
  tmem_st_wait();
}

template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_softmax(BwdBars& bar, const CrossParams& p, const BwdOut& out, uint32_t tmem, uint32_t smem, const float* tab, int warp, int lane) {
  using L = Bwd<kD>;
  constexpr bool kTwo = !kKeys || L::kTwoForKeys;
  const int w = warp >> 2, quarter = warp & 3, t = quarter * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16, mine = tmem + lanes + w * 32;
  volatile int* abort_flag = &bar.abort_flag;
  Ring<L::stages_a(kKeys)> ra;
  Ring<kTwo ? 2 : 1> rs;
  int it = 0, runs = 0;
  Ring<2> rt;
  for (; warp_ready(&bar.tasks.full[rt.stage], rt.parity, abort_flag, p.status, kStatusWaitFull); ++runs) {
    const volatile Task& task = bar.tasks.task[rt.stage];
    if (!task.valid) break;
    const int b = task.b, i0 = task.i0, i1 = task.i1;
    const bool stays_masked = kKeys && task.masked;
    // of the row: an entry of the mask, or statistics
    float2 entry = make_float2(0.f, 0.f);
    float neg_l = 0.f, neg_d = 0.f;
    if (kKeys) {
      if (stays_masked) entry = key_entry(p, b, task.at * 128 + t, task.base);
    } else if (task.at * 128 + t < p.R) {
      const long long row = (static_cast<long long>(b) * p.Hq + task.h) * p.R + task.at * 128 + t;
      neg_l = -__ldcg(out.stats + row);
      neg_d = -__ldcg(out.D + row);
    }
    int2 next = make_int2(0, stays_masked);
    if (!kKeys) next = live_block(p, b, i0);
    for (int i = i0; i < i1; ++i) {
      const bool masked = next.y;
      const int here = p.Sk - next.x * kKeys;        // keys of the block
      if (!kKeys && i + 1 < i1) next = live_block(p, b, i + 1);
      const float* tb = tab + ra.stage * 256 + (kKeys ? w * 32 : w * 64);
      const uint32_t tS = mine + (rs.stage ? (kKeys ? L::S2_KEYS : L::S2_ROWS) : L::S), tDP = mine + L::DP;
      if (!warp_ready(&bar.tab_full[ra.stage], ra.parity, abort_flag, p.status, kStatusWaitFull)) return;        // every turn: a parity tells only the last two apart
      if (!warp_ready_here(&bar.s_full[rs.stage], rs.parity, abort_flag, p.status, kStatusWaitAccum)) return;
      tc_fence_after_sync();
      if (masked) masked_scores<kKeys>(tS, entry, reinterpret_cast<const float2*>(tb));
      uint32_t pr[32];
      make_p<kKeys>(tS, masked ? 1.f : p.scale * kLog2e, tb, masked || kKeys ? neg_l : neg_l - task.base, pr);
      if (kKeys) {
        tmem_st_wait();
        tc_fence_before_sync();
        arrive_together(&bar.p_ready[rs.stage], lane);
      }
      if (!warp_ready_here(&bar.dp_full, it & 1, abort_flag, p.status, kStatusWaitAccum)) return;
      tc_fence_after_sync();
      if (masked) {
        masked_dp<kKeys>(tDP, entry, reinterpret_cast<const float2*>(tb));
        if (!kKeys && p.mask) {        // nor of an absent key's K, which its dS of zero meets: S and dP have been read from it
          if (w == 0 && t < here && reinterpret_cast<const float2*>(tb)[t].y == -INFINITY) zero_row<kD>(smem + L::RING + ra.stage * L::kTile, 128, t);
          fence_proxy_async_smem();
        }
      }
      make_ds<kKeys>(tDP, tb + 128, neg_d, pr);
      tmem_st_wait();
      tc_fence_before_sync();
      arrive_together(&bar.ds_ready, lane);
      ++it;
      ra.next();
      rs.next();
    }
    // ---- the run's sums. Keys: half of the warps write dK, the others dV; rows: all of them dQ
    if (!warp_ready(&bar.acc_done, runs & 1, abort_flag, p.status, kStatusWaitAccum)) return;
    tc_fence_after_sync();
    const int n = task.at * 128 + t, h = task.h;        // this thread's key or row
    const bool whole = task.whole, inside = kKeys ? n < p.Sk : n < p.R, is_v = kKeys && w >= 2;
    constexpr int kStep = kKeys ? kD / 2 : kD / 4;
    const int c0 = (kKeys ? w & 1 : w) * kStep;
    const uint32_t acc = tmem + (is_v ? L::ACC0 : L::ACC1) + lanes + c0;
    const float mul = is_v ? 1.f : p.scale;
    const bool absent = stays_masked && entry.y == -INFINITY;        // no gradient, whatever its probability of zero has met: a row's NaN or infinity is no number times zero
    float* part = nullptr;
    __nv_bfloat16* to = nullptr;
    if (!whole) {
      if (warp == 0 && lane == 0) bar.left[task.slot] = Left{1, task.ends, b, task.tile};
      const long long slot = kKeys ? (blockIdx.x * 2ll + task.slot) * 2 + is_v : (out.key_ctas + blockIdx.x) * 2ll + task.slot;
      part = out.part + (slot * 128 + t) * kD + c0;
    } else if (kKeys) {
      to = (is_v ? out.dv : out.dk) + b * out.ksb + n * out.kss + h * out.ksh + c0;
    } else {
      to = out_row(p, out.dq, out.qsb, out.qss, out.qsh, b, h, n) + c0;
    }
#pragma unroll 1
    for (int c = 0; c < kStep; c += 16) {
      uint32_t v[16];
      tmem_ld16(acc + c, v);
      tmem_ld_wait();
      float f[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        asm volatile("" : "+r"(v[e]));
        f[e] = absent ? 0.f : __uint_as_float(v[e]) * mul;
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(part + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
      } else if (inside) {
#pragma unroll
        for (int e = 0; e < 16; e += 8) *reinterpret_cast<uint4*>(to + c + e) = pack8(f + e);
      }
    }
    tc_fence_before_sync();
    arrive_warp(&bar.tasks.empty[rt.stage], lane);
    rt.next();
  }
}

template <int kD, bool kMany>
__global__ void __launch_bounds__(kBwdThreads, 1)
cross_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                 const CrossParams p, const BwdOut out) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using L = Bwd<kD>;
  static_assert(sizeof(BwdBars) <= 512, "barriers");
  BwdBars& bar = *reinterpret_cast<BwdBars*>(smem + L::BARS);
  float* tab = reinterpret_cast<float*>(smem + L::TAB);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const bool keys = static_cast<int>(blockIdx.x) < out.key_ctas;

  if (threadIdx.x == 0) {
    mbar_init(&bar.f_full, 1);
    mbar_init(&bar.f_empty, 1);
    for (int s = 0; s < 3; ++s) {
      mbar_init(&bar.a_full[s], 1);
      mbar_init(&bar.a_empty[s], 1);
      mbar_init(&bar.b_full[s], 1);
      mbar_init(&bar.b_empty[s], 1);
      mbar_init(&bar.tab_full[s], 1);
    }
    mbar_init(&bar.s_full[0], 1);
    mbar_init(&bar.s_full[1], 1);
    mbar_init(&bar.dp_full, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.p_ready[i], kBwdSoftmaxWarps);
    mbar_init(&bar.ds_ready, kBwdSoftmaxWarps);
    mbar_init(&bar.acc_done, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&bar.tasks.full[i], 1); mbar_init(&bar.tasks.empty[i], kBwdSoftmaxWarps + 2); }
    bar.left[0] = bar.left[1] = Left{0, 0, 0, 0};
    bar.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kBwdSoftmaxWarps) {
    tmem_alloc<1>(&bar.tmem_slot, 512);
    tmem_relinquish<1>();
  }
  if (warp == kBwdSoftmaxWarps + 1 && elect_one()) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bar.tmem_slot;
  pdl_entry();
  const uint32_t base = smem_u32(smem);

  if (warp == kBwdSoftmaxWarps + 1) {
    if (keys) bwd_loads<kD, true, kMany>(bar, p, out.keys, blockIdx.x, base, &tmK, &tmV, &tmQ, &tmDO);
    else bwd_loads<kD, false, kMany>(bar, p, out.rows, blockIdx.x - out.key_ctas, base, &tmQ, &tmDO, &tmK, &tmV);
  } else if (warp == kBwdSoftmaxWarps + 2) {
    if (keys) bwd_tables<kD, true>(bar, p, tab, out.stats, out.D, lane);
    else bwd_tables<kD, false>(bar, p, tab, out.stats, out.D, lane);
  } else if (warp == kBwdSoftmaxWarps) {
    if (keys) bwd_products<kD, true>(bar, p, tmem, base);
    else bwd_products<kD, false>(bar, p, tmem, base);
  } else {
    if (keys) bwd_softmax<kD, true>(bar, p, out, tmem, base, tab, warp, lane);
    else bwd_softmax<kD, false>(bar, p, out, tmem, base, tab, warp, lane);
    if (threadIdx.x == 0) {
      out.left[blockIdx.x * 2] = bar.left[0];
      out.left[blockIdx.x * 2 + 1] = bar.left[1];
    }
    if (p.live_count) {
      // what nothing streams past: blocks without a key, and the rows of batch rows without one, get zeros
      constexpr int kThreads = 32 * kBwdSoftmaxWarps, kVecs = kD / 8;
      for (long long x = blockIdx.x; x < static_cast<long long>(p.B) * p.key_blocks; x += gridDim.x) {
        const int b = static_cast<int>(x / p.key_blocks), i = static_cast<int>(x % p.key_blocks), n = live_of(p, b);
        if (i < n) continue;
        const int key0 = live_block(p, b, i).x * 128;
        for (int e = threadIdx.x; out.dk && e < 128 * p.Hk * kVecs; e += kThreads) {
          const int c = e % kVecs, h = e / kVecs % p.Hk, key = key0 + e / kVecs / p.Hk;
          if (key >= p.Sk) break;
          const long long at = b * out.ksb + key * out.kss + h * out.ksh + c * 8;
          *reinterpret_cast<uint4*>(out.dk + at) = *reinterpret_cast<uint4*>(out.dv + at) = make_uint4(0u, 0u, 0u, 0u);
        }
        if (n == 0 && i == 0 && out.dq)
          for (long long e = threadIdx.x; e < static_cast<long long>(p.Hq) * p.R * kVecs; e += kThreads) {
            const int c = static_cast<int>(e % kVecs), row = static_cast<int>(e / kVecs % p.R), h = static_cast<int>(e / kVecs / p.R);
            *reinterpret_cast<uint4*>(out_row(p, out.dq, out.qsb, out.qss, out.qsh, b, h, row) + c * 8) = make_uint4(0u, 0u, 0u, 0u);
          }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kBwdSoftmaxWarps) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, 512);
  }
}

// Before: D = rowsum(dO o), eight values a lane.
template <int kD>
__global__ void __launch_bounds__(256) cross_pre_kernel(const CrossParams p, const __nv_bfloat16* o, const long long osb, const long long oss, const long long osh,
                                                        const __nv_bfloat16* d_o, const long long gsb, const long long gss, const long long gsh,
                                                        float* D) {
  pdl_entry();
  const int lane = threadIdx.x & 31;
  constexpr int kLanes = kD / 8;
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.R;
  const int c = (threadIdx.x % kLanes) * 8;
  const unsigned m = kLanes == 16 ? 0xffffu << (lane & 16) : 0xffu << (lane & 24);
  for (long long row = (blockIdx.x * 256ll + threadIdx.x) / kLanes; row < rows; row += gridDim.x * 256ll / kLanes) {
    const int r = static_cast<int>(row % p.R), g = r & ((1 << p.pack_log2) - 1);
    const long long bh = row / p.R, b = bh / p.Hq, h = ((bh % p.Hq) << p.pack_log2) + g, s = r >> p.pack_log2;
    const uint4 x = *reinterpret_cast<const uint4*>(o + b * osb + s * oss + h * osh + c), y = *reinterpret_cast<const uint4*>(d_o + b * gsb + s * gss + h * gsh + c);
    float fx[8], fy[8], d = 0.f;
    VecIO<__nv_bfloat16>::unpack(x, fx);
    VecIO<__nv_bfloat16>::unpack(y, fy);
#pragma unroll
    for (int e = 0; e < 8; ++e) d += fx[e] * fy[e];
#pragma unroll
    for (int k = kLanes / 2; k > 0; k >>= 1) d += __shfl_xor_sync(m, d, k);
    if (c == 0) D[row] = d;
  }
}

// After: the stretches' shares of a tile added up in their order, by the block of the CTA that began it, four values a thread; keys: dK and dV.
template <int kD>
__global__ void __launch_bounds__(256) cross_sum_kernel(const CrossParams p, const BwdOut out, const int ctas) {
  __shared__ short with[kWith];
  __shared__ int count;
  pdl_entry();
  constexpr int kLanes = kD / 4;
  const int cta = blockIdx.x;
  const bool keys = cta < out.key_ctas;
  const Left first = out.left[cta * 2 + 1];
  if (!first.used || !FB_INDEX_OK(first.b, p.B, 304)) return;
  if (!FB_INDEX_OK(first.tile, keys ? static_cast<long long>(p.Hk) * live_of(p, first.b) : static_cast<long long>(p.Hq) * p.row_tiles, 305)) return;
  const int sharing = sharers(out.left, cta, keys ? out.key_ctas : ctas, with, &count);
  const int per = keys ? live_of(p, first.b) : p.row_tiles, h = first.tile / per, tile = first.tile - h * per;
  const int c = (threadIdx.x % kLanes) * 4, t = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes;
  const int n = (keys ? live_block(p, first.b, tile).x : tile) * 128 + t;
  if (n >= (keys ? p.Sk : p.R)) return;
  for (int v = 0; v < (keys ? 2 : 1); ++v) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < sharing; ++k) {
      const long long slot = keys ? (with[k] * 2ll + (k == 0)) * 2 + v : (out.key_ctas + with[k]) * 2ll + (k == 0);
      const float4 x = *reinterpret_cast<const float4*>(out.part + (slot * 128 + t) * kD + c);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    __nv_bfloat16* dst = keys ? (v ? out.dv : out.dk) + first.b * out.ksb + n * out.kss + h * out.ksh : out_row(p, out.dq, out.qsb, out.qss, out.qsh, first.b, h, n);
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2(acc.x, acc.y), pack2(acc.z, acc.w));
  }
}

// ------------------------------------------------------------------------------------------ host
int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }
long long round_up(long long n, long long m) { return (n + m - 1) / m * m; }

bool make_cross(const fb_cross_args& a, CrossParams& p, int& pack) {
  if (a.D != 64 && a.D != 128) return false;
  if (a.B < 1 || a.H < 1 || a.Hk < 1 || a.H % a.Hk || a.Sq < 1 || a.Sk < 1) return false;
  const int group = a.H / a.Hk;
  pack = group & -group;          // the largest power of two in it
  if (pack > 16) pack = 16;
  p.B = a.B;
  p.Hk = a.Hk;
  p.Hq = a.H / pack;
  p.per_kv = group / pack;
  p.pack_log2 = 31 - __builtin_clz(static_cast<unsigned>(pack));
  if (static_cast<long long>(a.Sq) * pack > 0x7fffff00ll || a.Sk > (1 << 30)) return false;
  p.R = a.Sq * pack;
  p.Sk = a.Sk;
  p.row_tiles = ceil_div(p.R, 128);
  p.key_blocks = ceil_div(p.Sk, kKeys);
  p.by_row_tiles = div_by(p.row_tiles);
  p.by_per_kv = div_by(p.per_kv);
  p.by_key_blocks = div_by(p.key_blocks);
  // tiles are counted in 32 bits, and so are the units of one for each CTA
  if (static_cast<long long>(p.B) * p.Hq * p.row_tiles > 0x3fffffffll || static_cast<long long>(p.B) * p.Hk * p.key_blocks > 0x3fffffffll ||
      static_cast<long long>(p.per_kv) * p.row_tiles > 0x7fffff || p.key_blocks > 0x7fffff)
    return false;
  p.mask = a.mask;
  p.mask_stride = a.mask_stride;
  p.mask_bool = a.mask_bool;
  p.scale = a.scale;
  p.table = !(a.scale > 0.f);
  p.status = a.status;
  if (a.mask) {
    p.live_count = a.mask_info;
    p.base = reinterpret_cast<float*>(a.mask_info + a.B);
    p.live = a.mask_info + 2ll * a.B;
    if (a.B > kScanned) p.before = p.live + static_cast<long long>(a.B) * p.key_blocks;
  }
  return true;
}

// CTAs for `units` of work over tiles of `length`, at most `most`, and whether their stretches hold whole tiles only. Tiles of up to four units are not cut: what is left of
// one costs about as much as a unit. Otherwise a stretch is two units at least.
Crew crew_of(const CrossParams& p, int tiles, int length, int most) {        // tiles of all batch rows, without a mask
  Crew c = {};
  if (most > kWith) most = kWith;
  c.whole = length <= 4 || most == 0;
  if (most == 0) return c;        // not wanted
  const long long units = static_cast<long long>(tiles) * length, n = c.whole ? tiles : (units + 1) / 2;
  c.ctas = static_cast<int>(n < most ? n : most);
  c.waves = tiles / c.ctas;
  c.first = c.waves * c.ctas;
  const long long rest = static_cast<long long>(tiles - c.first) * length;
  c.each = static_cast<int>(rest / c.ctas);
  c.more = static_cast<int>(rest % c.ctas);
  c.by_ctas = div_by(c.ctas);
  c.by_length = div_by(length);
  c.by_tiles = div_by(tiles / p.B);
  return c;
}
// A unit of keys takes four products and a unit of rows three: 2450 and 2070 cycles (heads of 64), 3400 and 2250 (128).
struct Crews {
  Crew rows, bwd_keys, bwd_rows;
};
// Whichever of the backward pass's gradients are not wanted leave the GPU to the others.
enum Wanted { kBoth, kRowsOnly, kKeysOnly };
Crews crews_of(const CrossParams& p, int D, Wanted wanted = kBoth) {
  const int row_tiles = p.B * p.Hq * p.row_tiles, sms = sm_count();
  const int most_keys = wanted == kRowsOnly ? 0 : wanted == kKeysOnly ? sms : D == 64 ? sms * 54 / 100 : sms * 60 / 100;
  return {crew_of(p, row_tiles, p.key_blocks, 2 * sms), crew_of(p, p.B * p.Hk * p.key_blocks, p.per_kv * p.row_tiles, most_keys), crew_of(p, row_tiles, p.key_blocks, sms - most_keys)};
}
// The forward pass's places in its workspace, in floats.
struct FwdSpace {
  long long ml, o, total;
};
// CTAs of a cluster to share a tile: as many as there is room for, of two blocks at least; 0 where tiles are short or many, or where a stretch would be so much
// shorter that it pays for its second launch (about as long as four units).
int parts_of(const CrossParams& p) {
  const long long tiles = static_cast<long long>(p.B) * p.Hq * p.row_tiles, slots = 2ll * sm_count();
  if (p.key_blocks <= 4 || tiles * 2 > slots) return 0;
  long long c = slots / tiles;
  if (c > p.key_blocks / 2) c = p.key_blocks / 2;
  if (c > 8) c = 8;        // (clusters of sixteen find room on few SMs at a time: 16 tiles of 256 blocks took 94 us against 62 in stretches)
  return ceil_div(p.key_blocks, c) > tiles * p.key_blocks / slots + 4 ? 0 : static_cast<int>(c);
}
FwdSpace space_fwd(const CrossParams& p, const Crew& c, int D) {
  FwdSpace f = {};
  if (c.whole || parts_of(p)) return f;
  f.ml = round_up(c.ctas * 2ll * 4, 32);
  f.o = f.ml + c.ctas * 2ll * 128 * 2;
  f.total = f.o + c.ctas * 2ll * 128 * D;
  return f;
}
struct BwdSpace {
  long long left, part, total;
};
BwdSpace space_bwd(const CrossParams& p, const Crews& c, int D) {
  BwdSpace f = {};
  f.left = round_up(static_cast<long long>(p.B) * p.Hq * p.R, 32);
  f.part = f.left + round_up((c.bwd_keys.ctas + c.bwd_rows.ctas) * 2ll * 4, 32);
  f.total = f.part + (c.bwd_keys.whole && c.bwd_rows.whole ? 0 : (c.bwd_keys.ctas * 4ll + c.bwd_rows.ctas * 2ll) * 128 * D);
  return f;
}

// What a mask comes to, for the 128-row kernels (`lists`), or its largest addends only.
cudaError_t look_through(const CrossParams& p, bool lists, cudaStream_t stream) {
  cudaError_t err = launch_pdl(cross_live_kernel, dim3(p.B), dim3(256), 0, stream, p);
  if (!err && lists && p.before) err = launch_pdl(cross_before_kernel, dim3(1), dim3(1024), 0, stream, p);
  return err;
}

// Like launch_pdl, in clusters.
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(void (*kern)(KArgs...), int blocks, int cluster, int threads, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// CTAs to share a tile of sixteen rows, 0 where tiles of 128 are better, and whether as a cluster. A warp has two chunks at least. A row more than
// sixteen makes the tensor cores' tile a better bargain as work grows: forward passes of B x H x Sq x Sk, D took, in tiles of sixteen and of 128 rows, with 2 x 12 x 64 x 200, 64
// (5 chunks an SM) 3.9 and 8.4 us, 3 x 12 x 77 x 1031, 64 (40) 11.7 and 13.0, 32 x 8 x 32 x 509, 64 (55) 13.2 and 17.2, 3 x 12 x 128 x 1031, 64 (64) 12.2 and 13.9, but 3 x 12 x 77 x 1031,
// 128 (79) 21.3 and 16.2, 32 x 8 x 64 x 509, 64 (111) 23.4 and 17.5. Up to sixteen rows these won at every size: 8 x 32 heads x 4 x 2000 on 8 key heads of 128 15.0 and 16.4,
// 64 x 32 heads x 1 x 1000 on 8 43.7 and 55.8, 128 x 16 x 1 x 500, 64 41.4 and 68.6, a single 1 x 8 x 1 x 1500, 64 4.8 and 9.2.
//
// With heads of 64 three CTAs fit an SM, with two stages to a warp's ring in place of three. That is better where there is work for the third (tokens of 16 x 8 over 1500 9.2 us against
// 10.1, 3 x 12 x 32 x 1031 8.7 and 11.3, 128 x 16 x 1 x 500 41.4 and 44.7), two better where there is not (4 x 8 x 4 x 2000 6.9 and 6.1, 3 x 12 x 128 x 1031 15.3 and 12.2).
struct FewShape {
  int parts, per_sm;
  bool cluster;
  long long ml, total;        // floats of workspace
};
FewShape few_shape(const CrossParams& p, int D) {
  FewShape f = {};
  const int chunks = ceil_div(p.Sk, 2048 / D);
  const long long tiles = static_cast<long long>(p.B) * p.Hq * ceil_div(p.R, 16);
  if (p.R > 16 && tiles * chunks > 70ll * sm_count()) return f;
  const auto parts_at = [&](int per_sm) {
    long long n = static_cast<long long>(per_sm) * sm_count() / tiles;
    if (n > ceil_div(chunks, 8)) n = ceil_div(chunks, 8);
    if (n > kWith) n = kWith;
    return n < 1 ? 1 : n;
  };
  f.per_sm = D == 64 && (tiles > 2ll * sm_count() || parts_at(3) > parts_at(2)) ? 3 : 2;
  const long long parts = parts_at(f.per_sm);
  f.cluster = parts <= 8;
  f.parts = static_cast<int>(parts);
  if (!f.cluster) {
    f.ml = round_up(tiles * parts * 16 * D, 32);
    f.total = f.ml + tiles * parts * 16 * 2;
  }
  return f;
}
template <int kD, int kPerSm>
int cross_few(const fb_cross_args& a, const CrossParams& p, const FewShape& shape, cudaStream_t stream) {
  if (shape.total && !a.workspace) return -3;
  FewArgs f = {};
  f.q = static_cast<const __nv_bfloat16*>(a.q);
  f.k = static_cast<const __nv_bfloat16*>(a.k);
  f.v = static_cast<const __nv_bfloat16*>(a.v);
  f.o = static_cast<__nv_bfloat16*>(a.o);
  for (int d = 0; d < 3; ++d) {
    f.qs[d] = a.q_strides[d];
    f.ks[d] = a.k_strides[d];
    f.vs[d] = a.v_strides[d];
    f.os[d] = a.o_strides[d];
  }
  f.stats = a.stats;
  f.parts = shape.parts;
  f.by_parts = div_by(f.parts);
  if (shape.total) {
    f.part_o = a.workspace;
    f.part_ml = reinterpret_cast<float2*>(a.workspace + shape.ml);
  }
  f.row_tiles = ceil_div(p.R, 16);
  f.by_rows = div_by(f.row_tiles);
  f.by_heads = div_by(p.Hq);
  if (p.mask && (a.stats || !p.mask_bool))        // the largest addends, and the lists for the backward pass
    if (const cudaError_t err = look_through(p, a.stats != nullptr, stream)) return static_cast<int>(err);
  constexpr auto kern = cross_few_kernel<kD, kPerSm>;
  constexpr int smem = Few<kD, kPerSm>::TOTAL, threads = Few<kD, kPerSm>::kWarps * 32;
  if (const cudaError_t err = allow_smem<kern>(smem, true)) return static_cast<int>(err);
  const int tiles = p.B * p.Hq * f.row_tiles, ctas = tiles * f.parts;
  cudaError_t err = f.parts > 1 && shape.cluster ? launch_clusters(kern, ctas, f.parts, threads, smem, stream, p, f)
                                                 : launch_pdl(kern, dim3(ctas), dim3(threads), static_cast<size_t>(smem), stream, p, f);
  if (!err && !shape.cluster) err = launch_pdl(cross_few_join_kernel<kD>, dim3(tiles, p.R < 16 ? p.R : 16), dim3(128), 0, stream, p, f);
  return static_cast<int>(err ? err : cudaGetLastError());
}

template <int kD, bool kMany>
int cross_fwd_tiles(const FwdOut& out, const CrossParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t stream) {
  constexpr auto kern = cross_fwd_kernel<kD, kMany>;
  constexpr int smem = Fwd<kD>::TOTAL + 1024;
  if (const cudaError_t err = allow_smem<kern>(smem, true)) return static_cast<int>(err);
  if (out.parts) {
    const int ctas = p.B * p.Hq * p.row_tiles * out.parts;
    if (const cudaError_t err = launch_clusters(kern, ctas, out.parts, kFwdThreads, smem, stream, tq, tk, tv, p, out)) return static_cast<int>(err);
    return static_cast<int>(cudaGetLastError());
  }
  return static_cast<int>(launch_pdl(kern, dim3(out.crew.ctas), dim3(kFwdThreads), static_cast<size_t>(smem), stream, tq, tk, tv, p, out));
}
template <int kD, bool kMany>
int cross_bwd_tiles(const BwdOut& out, const CrossParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tdo, cudaStream_t stream) {
  constexpr auto kern = cross_bwd_kernel<kD, kMany>;
  constexpr int smem = Bwd<kD>::TOTAL + 1024;
  if (const cudaError_t err = allow_smem<kern>(smem)) return static_cast<int>(err);
  return static_cast<int>(launch_pdl(kern, dim3(out.keys.ctas + out.rows.ctas), dim3(kBwdThreads), static_cast<size_t>(smem), stream, tq, tk, tv, tdo, p, out));
}

template <int kD>
int cross_fwd(const fb_cross_args& a, const CrossParams& p, int pack, cudaStream_t stream) {
  if (const FewShape shape = few_shape(p, kD); shape.parts) {
    if constexpr (kD == 64)
      if (shape.per_sm == 3) return cross_few<64, 3>(a, p, shape, stream);
    return cross_few<kD, 2>(a, p, shape, stream);
  }
  CUtensorMap tq, tk, tv;
  int e = make_tmap_rows(&tq, a.q, kD, pack, a.Sq, p.Hq, a.B, a.q_strides[0], a.q_strides[1], a.q_strides[2]);
  if (!e) e = make_tmap_rows(&tk, a.k, kD, 1, a.Sk, a.Hk, a.B, a.k_strides[0], a.k_strides[1], a.k_strides[2]);
  if (!e) e = make_tmap_rows(&tv, a.v, kD, 1, a.Sk, a.Hk, a.B, a.v_strides[0], a.v_strides[1], a.v_strides[2]);
  if (e) return e;
  const Crews crews = crews_of(p, kD);
  const FwdSpace f = space_fwd(p, crews.rows, kD);
  if (f.total && !a.workspace) return -3;
  FwdOut out = {};
  out.o = static_cast<__nv_bfloat16*>(a.o);
  out.osb = a.o_strides[0];
  out.oss = a.o_strides[1];
  out.osh = a.o_strides[2];
  out.stats = a.stats;
  out.crew = crews.rows;
  out.parts = parts_of(p);
  out.by_parts = div_by(out.parts ? out.parts : 1);
  if (f.total) {
    out.left = reinterpret_cast<Left*>(a.workspace);
    out.part_ml = reinterpret_cast<float2*>(a.workspace + f.ml);
    out.part_o = a.workspace + f.o;
  }
  if (p.mask)
    if (const cudaError_t err = look_through(p, true, stream)) return static_cast<int>(err);
  if (const int rc = p.before ? cross_fwd_tiles<kD, true>(out, p, tq, tk, tv, stream) : cross_fwd_tiles<kD, false>(out, p, tq, tk, tv, stream)) return rc;
  if (!out.parts && !out.crew.whole)
    if (const cudaError_t err = launch_pdl(cross_join_kernel<kD>, dim3(out.crew.ctas, ceil_div((p.R < 128 ? p.R : 128) * kD, 1024)), dim3(256), 0, stream, p, out, out.crew.ctas)) return static_cast<int>(err);
  return static_cast<int>(cudaGetLastError());
}

template <int kD>
int cross_bwd(const fb_cross_args& a, const CrossParams& p, int pack, cudaStream_t stream) {
  CUtensorMap tq, tk, tv, tdo;
  int e = make_tmap_rows(&tq, a.q, kD, pack, a.Sq, p.Hq, a.B, a.q_strides[0], a.q_strides[1], a.q_strides[2]);
  if (!e) e = make_tmap_rows(&tk, a.k, kD, 1, a.Sk, a.Hk, a.B, a.k_strides[0], a.k_strides[1], a.k_strides[2]);
  if (!e) e = make_tmap_rows(&tv, a.v, kD, 1, a.Sk, a.Hk, a.B, a.v_strides[0], a.v_strides[1], a.v_strides[2]);
  if (!e) e = make_tmap_rows(&tdo, a.d_o, kD, pack, a.Sq, p.Hq, a.B, a.do_strides[0], a.do_strides[1], a.do_strides[2]);
  if (e) return e;
  const Crews crews = crews_of(p, kD, !a.dk ? kRowsOnly : !a.dq ? kKeysOnly : kBoth);
  const BwdSpace f = space_bwd(p, crews, kD);
  BwdOut out = {};
  float* D = a.workspace;
  out.stats = a.stats;
  out.D = D;
  out.left = reinterpret_cast<Left*>(a.workspace + f.left);
  out.part = a.workspace + f.part;
  out.dq = static_cast<__nv_bfloat16*>(a.dq);
  out.dk = static_cast<__nv_bfloat16*>(a.dk);
  out.dv = static_cast<__nv_bfloat16*>(a.dv);
  out.qsb = a.dq_strides[0]; out.qss = a.dq_strides[1]; out.qsh = a.dq_strides[2];
  out.ksb = a.dk_strides[0]; out.kss = a.dk_strides[1]; out.ksh = a.dk_strides[2];
  out.keys = crews.bwd_keys;
  out.rows = crews.bwd_rows;
  out.key_ctas = out.keys.ctas;
  const long long want = (static_cast<long long>(p.B) * p.Hq * p.R * (kD / 8) + 255) / 256, most = 16ll * sm_count();
  if (const cudaError_t err = launch_pdl(cross_pre_kernel<kD>, dim3(static_cast<unsigned>(want < most ? want : most)), dim3(256), 0, stream, p, static_cast<const __nv_bfloat16*>(a.o), a.o_strides[0],
                                         a.o_strides[1], a.o_strides[2], static_cast<const __nv_bfloat16*>(a.d_o), a.do_strides[0], a.do_strides[1], a.do_strides[2], D))
    return static_cast<int>(err);
  const int ctas = out.keys.ctas + out.rows.ctas;
  if (const int rc = p.before ? cross_bwd_tiles<kD, true>(out, p, tq, tk, tv, tdo, stream) : cross_bwd_tiles<kD, false>(out, p, tq, tk, tv, tdo, stream)) return rc;
  if (!out.keys.whole || !out.rows.whole)
    if (const cudaError_t err = launch_pdl(cross_sum_kernel<kD>, dim3(ctas, kD / 8), dim3(256), 0, stream, p, out, ctas)) return static_cast<int>(err);
  return static_cast<int>(cudaGetLastError());
}

bool rows_ok(const void* p, const long long* st) { return p && strides_ok(p, st[0], st[1], st[2]); }
bool aside_ok(const fb_cross_args& a) {
  return (!a.mask || (a.mask_info && (a.mask_bool || aligned(a.mask, 4)))) && aligned(a.mask_info, 4) && aligned(a.stats, 4) && aligned(a.workspace, 16) && aligned(a.status, 4);
}

}  // namespace
}  // namespace fb

extern "C" long long fb_cross_workspace(const fb_cross_args* args, int backward) {
  using namespace fb;
  if (!args) return -3;
  CrossParams p = {};
  int pack;
  if (!make_cross(*args, p, pack)) return -4;
  const Crews crews = crews_of(p, args->D);
  if (backward) {        // of whichever gradients the call will want
    long long most = 0;
    for (const Wanted w : {kBoth, kRowsOnly, kKeysOnly})
      if (const long long n = space_bwd(p, crews_of(p, args->D, w), args->D).total; n > most) most = n;
    return most;
  }
  return few_shape(p, args->D).parts ? few_shape(p, args->D).total : space_fwd(p, crews.rows, args->D).total;
}
extern "C" long long fb_cross_mask_info(const fb_cross_args* args) {
  using namespace fb;
  if (!args) return -3;
  CrossParams p = {};
  int pack;
  if (!make_cross(*args, p, pack)) return -4;
  if (!p.mask) return 0;
  return p.B * (2ll + p.key_blocks) + (p.B > kScanned ? 2 * (p.B + 1ll) : 0);
}

extern "C" int fb_cross_attn_fwd(const fb_cross_args* args, void* stream) {
  using namespace fb;
  if (!args) return -3;
  const fb_cross_args& a = *args;
  CrossParams p = {};
  int pack;
  if (!make_cross(a, p, pack)) return -4;
  if (!rows_ok(a.q, a.q_strides) || !rows_ok(a.k, a.k_strides) || !rows_ok(a.v, a.v_strides) || !rows_ok(a.o, a.o_strides) || !aside_ok(a)) return -3;
  const auto s = static_cast<cudaStream_t>(stream);
  return a.D == 64 ? cross_fwd<64>(a, p, pack, s) : cross_fwd<128>(a, p, pack, s);
}

extern "C" int fb_cross_attn_bwd(const fb_cross_args* args, void* stream) {
  using namespace fb;
  if (!args) return -3;
  const fb_cross_args& a = *args;
  CrossParams p = {};
  int pack;
  if (!make_cross(a, p, pack)) return -4;
  if (!rows_ok(a.q, a.q_strides) || !rows_ok(a.k, a.k_strides) || !rows_ok(a.v, a.v_strides) || !rows_ok(a.o, a.o_strides) || !rows_ok(a.d_o, a.do_strides) ||
      (a.dq && !rows_ok(a.dq, a.dq_strides)) || (a.dk && !rows_ok(a.dk, a.dk_strides)) || (a.dv && !rows_ok(a.dv, a.dk_strides)) || !aside_ok(a) || !a.stats ||
      !a.workspace)
    return -3;
  if (!a.dk != !a.dv || (!a.dq && !a.dk)) return -3;
  const auto s = static_cast<cudaStream_t>(stream);
  return a.D == 64 ? cross_bwd<64>(a, p, pack, s) : cross_bwd<128>(a, p, pack, s);
}

FB_BOUNDS_ATTACH(cross_attn)
