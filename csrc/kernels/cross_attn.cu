// Attention of queries over keys and values of another length (an encoder's states), forward and backward, head dim 64 and 128, on tcgen05.
//
//   o = softmax(scale q k^T + mask) v;   P from the saved row statistics:   dV = P^T dO,   dS = P (dO V^T - D),   D = rowsum(dO o),   dQ = scale dS K,   dK = scale dS^T Q
//
// Rows. The query heads of a key head lie side by side in memory, so a tile's rows are (query, head) pairs of a power of two `pack` of them, head fastest, which one 5-D
// tensor map gives; what is left of the group is heads of their own. One key head's K and V are so read once for all of them, and few queries fill a tile better.
//
// Masks are of keys. Blocks of 128 keys none of which takes part are left out; blocks all of which do, with nothing added, take the short path; the rest go by a table
// of {scale, addend} for each key. A key at -inf is absent: its score is replaced whatever it is, and where it meets a product as a row of the streamed operand that row
// is zeroed in shared memory, so infinities and NaN behind a mask reach nothing. An addend beyond 2^100 takes the score's place, as it would in 64 bits.
// Addends are taken relative to the batch row's largest, so that a mask common to a row's keys costs its scores no bits.
//
// Statistics, sums and products are fp32; P and dS are rounded to bf16 once, as operands of the tensor cores.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../include/flodl_b200.h"
#include "flash_attn_common.cuh"

namespace fb {
namespace {

constexpr int kKeys = 128;          // keys of a mask block
constexpr int kMaxBlocks = 4096;    // mask blocks of one work item
constexpr float kHuge = 1.2676506e30f;      // 2^100

struct CrossParams {
  int B, Hq, Hk, R, Sk;             // Hq = H / pack rows of heads; R = Sq * pack rows each
  int pack_log2, per_kv;            // log2 of pack; rows of heads that share a key head
  const void* mask;                 // [B, Sk]: one byte a key (0: absent), or fp32 addends; null: none
  float* base;                      // [B] of addends: the batch row's largest, which the forward pass leaves for the backward pass (null: nobody wants it)
  long long mask_stride;
  int mask_bool;
  float scale;
  int table;                        // 1: every block by the table (the short path wants a positive scale)
  int* status;
};

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
    const int kv = blk * kKeys + i * 32 + lane;
    bool in = kv < p.Sk, plain = in;
    if (in && p.mask) {
      const long long at = b * p.mask_stride + kv;
      if (p.mask_bool) {
        in = plain = static_cast<const uint8_t*>(p.mask)[at] != 0;
      } else {
        const float a = static_cast<const float*>(p.mask)[at];
        in = a != -INFINITY;
        plain = a == 0.f;
      }
    }
    any |= in;
    all &= plain;
  }
  any = __any_sync(0xffffffffu, any);
  all = __all_sync(0xffffffffu, all);
  return !any ? 0 : all && !p.table ? 2 : 1;
}
__device__ __forceinline__ int block_state_unmasked(const CrossParams& p, int blk) { return (blk + 1) * kKeys <= p.Sk && !p.table ? 2 : 1; }

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

// Waits, whatever the block's state, until the copies counted by `bar` have landed: shared memory may not be left while one is on its way to it.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  for (uint32_t it = 0; it < (1u << 20) && !mbar_test(bar, parity); ++it) __nanosleep(20);
}

// A whole warp's wait. Most find the phase already over, and a plain test says so in a quarter of the time (26 cycles against 98 of the waiting loop).
__device__ __forceinline__ bool warp_ready(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
  return warp_wait(bar, parity, abort_flag, status, code);
}

__device__ __forceinline__ uint64_t k_desc(uint32_t base, int bytes) { return desc_of(smem_desc_lo(base, 16) + (bytes >> 4), smem_desc_hi(1024)); }
__device__ __forceinline__ uint64_t mn_desc(uint32_t base, int bytes, int lbo) { return desc_of(smem_desc_lo(base, lbo) + (bytes >> 4), smem_desc_hi(1024)); }

// ===================================================================================== forward
// One CTA per 128 rows of a row of heads, and per part of the keys where there are few such tiles; two CTAs an SM, so that one's products run under the other's
// exponentials. Four softmax warps (a thread is a row), one that issues products, one that loads. P goes to the second product through TMEM.
constexpr int kFwdThreads = 192;
constexpr float kSlack = 8.f;       // the accumulator is scaled anew once a row's maximum has grown by 2^8: most blocks' maxima grow a little in some row of a warp

template <int kD>
struct Fwd {
  static constexpr int kStages = kD == 64 ? 2 : 1;
  static constexpr int kTile = 128 * kD * 2;
  static constexpr int Q = 0;
  static constexpr int K = Q + kTile;
  static constexpr int V = K + kStages * kTile;
  static constexpr int TAB = V + kStages * kTile;        // 2 x 128 x {scale, addend}
  static constexpr int BARS = TAB + 2 * 128 * 8;
  static constexpr int BASE = BARS + 160;                // 6 floats: the warps' largest addends
  static constexpr int STATE = BARS + 256;               // a byte for each of the item's blocks
  static constexpr int bytes(int blocks) { return STATE + (blocks + 15) / 16 * 16 + 1024; }
  // Columns of TMEM. With 128 values a head P takes the place of the scores, which it is made from.
  static constexpr uint32_t S = 0, P = kD == 64 ? 128 : 0, O = kD == 64 ? 192 : 128;
};

struct FwdOut {
  __nv_bfloat16* o;
  long long osb, oss, osh;
  float* stats;                // [B, Hq, R] log2 of the sum of the exponentials, relative to the mask's base; null: not wanted
  float* part_o;               // parts > 1: [parts][B, Hq, R][D] sums relative to the part's maximum
  float2* part_ml;             // ... {maximum, sum}
  int parts, blocks_per_part, n_tiles;
};

__device__ __forceinline__ __nv_bfloat16* out_row(const CrossParams& p, __nv_bfloat16* base, long long sb, long long ss, long long sh, int b, int h, int r) {
  const int g = r & ((1 << p.pack_log2) - 1);
  return base + b * sb + (r >> p.pack_log2) * ss + ((static_cast<long long>(h) << p.pack_log2) + g) * sh;
}

template <int kD>
__global__ void __launch_bounds__(kFwdThreads, 2)
cross_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CrossParams p, const FwdOut out) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using L = Fwd<kD>;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;     // [kStages]
  uint64_t* k_empty = bars + 3;
  uint64_t* v_full = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;     // the scores of a block are in TMEM
  uint64_t* s_free = bars + 10;    // ... and in the softmax warps' registers
  uint64_t* p_ready = bars + 11;   // the probabilities are in TMEM and O has been rescaled where it had to be
  uint64_t* pv_done = bars + 12;   // P V has been added to O
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* tab = reinterpret_cast<float2*>(smem + L::TAB);
  uint8_t* state = smem + L::STATE;

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  int lin = blockIdx.x;
  const int part = lin % out.parts;
  lin /= out.parts;
  const int tile = lin % out.n_tiles;
  lin /= out.n_tiles;
  const int h = lin % p.Hq, b = lin / p.Hq, hk = h / p.per_kv;
  const int row0 = tile * 128, rows = min(128, p.R - row0);
  const int j0 = part * out.blocks_per_part, n_blocks = min(out.blocks_per_part, (p.Sk + kKeys - 1) / kKeys - j0);
  const int warps = (rows + 31) >> 5;        // softmax warps that have rows

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < L::kStages; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    mbar_init(s_full, 1);
    mbar_init(s_free, warps);
    mbar_init(p_ready, warps);
    mbar_init(pv_done, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == 4) {
    tmem_alloc<1>(tmem_slot, 256);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_entry();       // behind the allocation: the next kernel's may not come before it
  for (int j = warp; j < n_blocks; j += kFwdThreads / 32) {
    const int s = p.mask ? block_state(p, b, j0 + j, lane) : block_state_unmasked(p, j0 + j);
    if (lane == 0) state[j] = static_cast<uint8_t>(s);
  }
  float* bases = reinterpret_cast<float*>(smem + L::BASE);
  const bool addends = p.mask && !p.mask_bool;
  if (addends) {
    float a = -INFINITY;
    for (int kv = threadIdx.x; kv < p.Sk; kv += kFwdThreads) a = fmaxf(a, key_addend(p, b, kv));
    a = warp_max(a);
    if (lane == 0) bases[warp] = a;
  }
  __syncthreads();
  float base = 0.f;
  if (addends) {
    base = max3(max3(bases[0], bases[1], bases[2]), bases[3], fmaxf(bases[4], bases[5]));
    if (isinf(base)) base = 0.f;       // no key takes part
    if (p.base && threadIdx.x == 0) p.base[b] = base;       // every CTA of the batch row the same
  }
  const uint32_t sQ = smem_u32(smem + L::Q), sK = smem_u32(smem + L::K), sV = smem_u32(smem + L::V);

  if (warp == 5) {
    // ------------------------------------------------------------------ loads
    if (elect_one()) {
      mbar_expect_tx(q_full, L::kTile);
      load_tile<kD>(sQ, &tmQ, q_full, 128, row0 >> p.pack_log2, h, b);
    }
    __syncwarp();
    int it = 0, ks = 0, vs = 0;
    for (int j = 0; j < n_blocks; ++j) {
      if (!state[j]) continue;
      const int st = it % L::kStages;
      const uint32_t ph = ((it / L::kStages) & 1) ^ 1;
      if (!warp_ready(&k_empty[st], ph, abort_flag, p.status, kStatusWaitEmpty)) break;
      if (elect_one()) {
        mbar_expect_tx(&k_full[st], L::kTile);
        load_tile<kD>(sK + st * L::kTile, &tmK, &k_full[st], 128, (j0 + j) * kKeys, hk, b);
      }
      __syncwarp();
      ++ks;
      if (!warp_ready(&v_empty[st], ph, abort_flag, p.status, kStatusWaitEmpty)) break;
      if (elect_one()) {
        mbar_expect_tx(&v_full[st], L::kTile);
        load_tile<kD>(sV + st * L::kTile, &tmV, &v_full[st], 128, (j0 + j) * kKeys, hk, b);
      }
      __syncwarp();
      ++vs;
      ++it;
    }
    drain(q_full, 0);
    for (int u = max(0, ks - L::kStages); u < ks; ++u) drain(&k_full[u % L::kStages], (u / L::kStages) & 1);
    for (int u = max(0, vs - L::kStages); u < vs; ++u) drain(&v_full[u % L::kStages], (u / L::kStages) & 1);
  } else if (warp == 4) {
    // ------------------------------------------------------------------ products
    const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0), idesc_o = make_idesc_bf16(128, kD, 0, 1);
    int n = 0;
    for (int j = 0; j < n_blocks; ++j) n += state[j] != 0;
    auto scores = [&](int it) {
      const int st = it % L::kStages;
      if (!warp_ready(&k_full[st], (it / L::kStages) & 1, abort_flag, p.status, kStatusWaitFull)) return false;
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kD / 16; ++k)
          umma_bf16<1>(tmem + L::S, k_desc(sQ, (k >> 2) * 16384 + (k & 3) * 32), k_desc(sK + st * L::kTile, (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
        umma_commit(s_full);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool ok = n > 0 && warp_ready(q_full, 0, abort_flag, p.status, kStatusWaitFull) && scores(0);
    for (int it = 0; it < n && ok; ++it) {
      if (kD == 64 && it + 1 < n) {        // P has a place of its own: the next scores may come under this block's exponentials
        ok = warp_ready(s_free, it & 1, abort_flag, p.status, kStatusWaitEpi) && scores(it + 1);
        if (!ok) break;
      }
      const int st = it % L::kStages;
      ok = warp_ready(p_ready, it & 1, abort_flag, p.status, kStatusWaitEpi) && warp_ready(&v_full[st], (it / L::kStages) & 1, abort_flag, p.status, kStatusWaitFull);
      if (!ok) break;
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 128 / 16; ++k) umma_bf16_ts(tmem + L::O, tmem + L::P + k * 8, mn_desc(sV + st * L::kTile, k * 2048, 16384), idesc_o, it > 0 || k > 0);
        umma_commit(pv_done);
        umma_commit(&v_empty[st]);
      }
      __syncwarp();
      if (kD != 64 && it + 1 < n) ok = warp_ready(pv_done, it & 1, abort_flag, p.status, kStatusWaitAccum) && scores(it + 1);
    }
  } else if (warp < warps) {
    // ------------------------------------------------------------------ softmax: a thread is a row
    const int t = threadIdx.x, r = row0 + t;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const float sc = p.scale * kLog2e;
    float m = -INFINITY, l = 0.f;       // the maximum the accumulator is relative to, and the sum
    bool ok = true;
    int it = 0;
    // After a wait that gave up the loop runs out without work, so that no warp is missed at the barriers.
    for (int j = 0; j < n_blocks; ++j) {
      const int kind = state[j];
      if (!kind) continue;
      float2* tb = tab + (it & 1) * 128;
      if (kind == 1) {
        for (int e = t; e < kKeys; e += warps * 32) {
          const float2 k = key_entry(p, b, (j0 + j) * kKeys + e, base);
          tb[e] = k;
          if (p.mask && k.y == -INFINITY && ok) {        // an absent key's values meet a probability of zero
            ok = mbar_wait(&v_full[it % L::kStages], (it / L::kStages) & 1, abort_flag, p.status, kStatusWaitFull);
            if (ok) zero_row<kD>(sV + (it % L::kStages) * L::kTile, 128, e);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        fence_proxy_async_smem();
        asm volatile("bar.sync 1, %0;" ::"r"(warps * 32) : "memory");
      }
      ok = ok && warp_ready(s_full, it & 1, abort_flag, p.status, kStatusWaitAccum);
      if (ok) {
        tc_fence_after_sync();
        if (kind != 2) apply_table<4>(tmem + L::S + lanes, tb);        // from here on all blocks are alike
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tmem + L::S + lanes + 32 * c, s[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(s[c][i]));
        if (kD == 64) {
          tc_fence_before_sync();
          arrive_warp(s_free, lane);
        }
        const float mul = kind == 2 ? sc : 1.f, below = kind == 2 ? base : 0.f;        // a key with nothing added is `base` below the largest
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
        const float m_new = fmaxf(m, fmaf(mul, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), -below));
        if (it > 0) {        // P may be overwritten, O touched
          ok = warp_ready(pv_done, (it - 1) & 1, abort_flag, p.status, kStatusWaitAccum);
          tc_fence_after_sync();
          // (m is -inf where no key has been seen: its sums are zeros, and stay so whatever they are scaled by)
          if (ok && __any_sync(0xffffffffu, m_new > m + kSlack)) {
            const float alpha = m_new == -INFINITY ? 1.f : ex2_approx(m - m_new);
            m = m_new;
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < kD; c += 16) {
              uint32_t v[16];
              tmem_ld16(tmem + L::O + lanes + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st16(tmem + L::O + lanes + c, v);
            }
          }
        }
        if (ok) {
          if (it == 0) m = m_new;
          const float neg_m = m == -INFINITY ? 0.f : -m - below;
          F2 sum[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float lo, hi;
              f2_get(f2_fma(f2_make(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), f2_splat(mul), f2_splat(neg_m)), lo, hi);
              lo = ex2_approx(lo);
              hi = ex2_approx(hi);
              sum[(i >> 1) & 1] = f2_add(sum[(i >> 1) & 1], f2_make(lo, hi));
              pk[i >> 1] = pack2(lo, hi);
            }
            tmem_st16(tmem + L::P + lanes + 16 * c, pk);
          }
          float a0, a1, b0, b1;
          f2_get(sum[0], a0, a1);
          f2_get(sum[1], b0, b1);
          l += (a0 + a1) + (b0 + b1);
          tmem_st_wait();
          tc_fence_before_sync();
          arrive_warp(p_ready, lane);
        }
      }
      ++it;
    }
    ok = __all_sync(0xffffffffu, ok && (it > 0 ? mbar_wait(pv_done, (it - 1) & 1, abort_flag, p.status, kStatusWaitAccum)
                                               : mbar_wait(q_full, 0, abort_flag, p.status, kStatusWaitFull)));        // Q's place is written below
    if (ok) {
      tc_fence_after_sync();
      const long long at = (static_cast<long long>(b) * p.Hq + h) * p.R + r;
      const bool split = out.parts > 1;
      const float inv = split ? 1.f : l == 0.f ? 0.f : 1.f / l;
      if (t < rows) {
        const long long pat = static_cast<long long>(part) * p.B * p.Hq * p.R + at;
        if (split) out.part_ml[pat] = make_float2(m, l);
        // a row that no key takes part in: +inf, which makes every probability 2^-inf = 0
        else if (out.stats) out.stats[at] = l == 0.f ? INFINITY : m + log2f(l);
      }
      float* po = split ? out.part_o + (static_cast<long long>(part) * p.B * p.Hq * p.R + at) * kD : nullptr;
#pragma unroll
      for (int c0 = 0; c0 < kD; c0 += 32) {
        uint32_t v[32];
        if (it > 0) {
          tmem_ld32_sync(tmem + L::O + lanes + c0, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]) * inv;
        if (split) {
          if (t < rows)
#pragma unroll
            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(po + c0 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
        } else {       // through the warp's 4 KB of each of Q's panels, which every product has read
          stage_half(sQ + (c0 >> 6) * 16384 + warp * 4096, lane, c0 & 32, f);
        }
      }
      if (!split) {
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
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem, 256);
  }
}

// The parts of a row joined: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i. A warp takes 128 / kD rows at a time, four values a lane.
template <int kD>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossParams p, const FwdOut out) {
  pdl_entry();
  constexpr int kLanes = kD / 4;
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.R;
  const int c = (threadIdx.x % kLanes) * 4;
  for (long long row = (blockIdx.x * 256ll + threadIdx.x) / kLanes; row < rows; row += gridDim.x * 256ll / kLanes) {
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < out.parts; ++i) m = fmaxf(m, out.part_ml[i * rows + row].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < out.parts; ++i) {
      const float2 ml = out.part_ml[i * rows + row];
      const float4 v = *reinterpret_cast<const float4*>(out.part_o + (i * rows + row) * kD + c);
      const float w = ex2_approx(ml.x - ref);
      l += w * ml.y;
      acc.x += w * v.x; acc.y += w * v.y; acc.z += w * v.z; acc.w += w * v.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int r = static_cast<int>(row % p.R);
    const long long bh = row / p.R;
    __nv_bfloat16* dst = out_row(p, out.o, out.osb, out.oss, out.osh, static_cast<int>(bh / p.Hq), static_cast<int>(bh % p.Hq), r) + c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(acc.x * inv, acc.y * inv), pack2(acc.z * inv, acc.w * inv));
    if (out.stats && c == 0) out.stats[row] = l == 0.f ? INFINITY : m + log2f(l);
  }
}

// ==================================================================================== backward
// Two kinds of work item, in one launch. Both keep a tile of 128 rows of two tensors in shared memory and stream tiles of 128 rows of the other two:
//   keys:  K, V stay; Q, dO stream.   S^T = K Q^T, dP^T = V dO^T;   dV += P^T dO,  dK += dS^T Q
//   rows:  Q, dO stay; K, V stream.   S = Q K^T,   dP = dO V^T;     dQ += dS K
// Scores are so worked out twice, but P and dS reach their products in TMEM, in the place of the scores and the dP that they are made from, and never through shared memory,
// and every gradient is summed by one CTA in the order of the tiles: two calls give the same bits, with no atomics and no pass over a scratch. Sixteen softmax
// warps: a thread is a row of the tile that stays and 32 of the streamed tile's columns. (With eight, 64 columns each, a warp's exponentials alone took 1050 cycles where the
// unit needs 512: two warps a scheduler do not hide the latencies.) Products of one CTA run in the order in which they are issued, so that what overwrites a place may be
// issued right behind what reads it: S(j+1) behind dV(j) (ahead of time, where there is a second buffer), dP(j+1) behind dK(j) or dQ(j).
// Tiles of 128 columns, not two of 64: with both operands in shared memory a product of 128 x 64 x 16 takes the 64 cycles of one of 128 x 128 x 16.
// Where there are few items, the streamed tiles are cut into parts, whose fp32 sums are added in their order by a second launch.
constexpr int kBwdSoftmaxWarps = 16;
constexpr int kBwdThreads = 32 * (kBwdSoftmaxWarps + 3);        // ... one that issues products, one that loads, one that fills tables

template <int kD>
struct Bwd {
  // Streamed tiles that are there at a time: of Q or K (A), of dO or V (B). A block of V has done its work with dP, Q, K and dO are read again by the products behind.
  static constexpr int stages_a(bool keys) { return kD == 64 ? 3 : keys ? 2 : 3; }
  static constexpr int stages_b(bool keys) { return kD == 64 ? 3 : keys ? 2 : 1; }
  static constexpr int kTile = 128 * kD * 2;
  static constexpr int F0 = 0, F1 = kTile;
  static constexpr int RING = 2 * kTile;                           // A's tiles, then B's
  static constexpr int TAB = RING + (kD == 64 ? 6 : 4) * kTile;    // 3 x 256 floats
  static constexpr int BARS = TAB + 3 * 1024;
  static constexpr int TOTAL = BARS + 256;
  // Columns of TMEM: one more buffer of scores where the accumulators leave room for it.
  static constexpr uint32_t S = 0, DP = 128, ACC0 = 256, ACC1 = 256 + kD;
  static constexpr uint32_t S2_KEYS = 384, S2_ROWS = kD == 64 ? 384 : 256;
  static constexpr bool kTwoForKeys = kD == 64;
};
static_assert(Bwd<128>::TOTAL + 1024 <= 227 * 1024, "shared memory budget");

struct BwdOut {
  const float* stats;              // of the forward pass
  const float* D;                  // [B, Hq, R]
  const uint8_t* state;            // [B, blocks] of a mask; null without one
  __nv_bfloat16 *dq, *dk, *dv;
  long long qsb, qss, qsh, ksb, kss, ksh;
  float *part_q, *part_k, *part_v; // [parts][B, Hq, R][D]; [parts][B, Hk, Sk][D]
  int parts_q, parts_k;            // parts of an item of rows, of keys
  int row_tiles, key_blocks;       // items of a row of heads, of a key head
  int key_items;                   // the first of all
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
  uint64_t f_full;
  uint64_t a_full[3], a_empty[3];     // a streamed tile of Q or K has landed; every product that reads it has retired
  uint64_t b_full[3], b_empty[3];     // ... of dO or V
  uint64_t tab_full[3];               // A's table is written
  uint64_t s_full[2], dp_full;        // scores and dP are in TMEM
  uint64_t p_ready, ds_ready;         // ... and P and dS in their place
  uint64_t acc_done;                  // every product has retired
  uint32_t tmem_slot;
  int abort_flag;
};

template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_products(BwdBars& bar, int* status, uint32_t tmem, uint32_t smem, int n) {
  using L = Bwd<kD>;
  volatile int* abort_flag = &bar.abort_flag;
  constexpr bool kTwo = !kKeys || L::kTwoForKeys;
  constexpr int kA = L::stages_a(kKeys), kB = L::stages_b(kKeys);
  const uint32_t idesc_s = make_idesc_bf16(128, 128, 0, 0), idesc_acc = make_idesc_bf16(128, kD, 0, 1);
  const auto s_at = [&](int it) { return tmem + (kTwo && (it & 1) ? (kKeys ? L::S2_KEYS : L::S2_ROWS) : L::S); };
  const auto a_at = [&](int it) { return smem + L::RING + it % kA * L::kTile; };
  const auto b_at = [&](int it) { return smem + L::RING + (kA + it % kB) * L::kTile; };
  const auto scores = [&](int it) {
    if (!warp_ready(&bar.a_full[it % kA], (it / kA) & 1, abort_flag, status, kStatusWaitFull)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kD / 16; ++k)
        umma_bf16<1>(s_at(it), k_desc(smem + L::F0, (k >> 2) * 16384 + (k & 3) * 32), k_desc(a_at(it), (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
      umma_commit(&bar.s_full[kTwo ? it & 1 : 0]);
    }
    __syncwarp();
    return true;
  };
  const auto dp = [&](int it) {
    if (!warp_ready(&bar.b_full[it % kB], (it / kB) & 1, abort_flag, status, kStatusWaitFull)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < kD / 16; ++k)
        umma_bf16<1>(tmem + L::DP, k_desc(smem + L::F1, (k >> 2) * 16384 + (k & 3) * 32), k_desc(b_at(it), (k >> 2) * 16384 + (k & 3) * 32), idesc_s, k > 0);
      umma_commit(&bar.dp_full);
      if (!kKeys) umma_commit(&bar.b_empty[it % kB]);
    }
    __syncwarp();
    return true;
  };
  // acc += (the 128 columns, each 32 left as bf16 in the first half of their place) x (the 128 rows of a streamed tile)
  const auto accumulate = [&](uint32_t acc, uint32_t from, uint32_t tile, int it, uint64_t* ready, uint64_t* empty) {
    if (!warp_ready(ready, it & 1, abort_flag, status, kStatusWaitEpi)) return false;
    tc_fence_after_sync();
    if (elect_one()) {
#pragma unroll
      for (int k = 0; k < 8; ++k) umma_bf16_ts(tmem + acc, from + (k >> 1) * 32 + (k & 1) * 8, mn_desc(tile, k * 2048, 16384), idesc_acc, it > 0 || k > 0);
      umma_commit(empty);
    }
    __syncwarp();
    return true;
  };
  bool ok = n > 0 && warp_ready(&bar.f_full, 0, abort_flag, status, kStatusWaitFull) && scores(0) && dp(0);
  for (int it = 0; it < n && ok; ++it) {
    const bool more = it + 1 < n;
    if (kTwo && more) ok = scores(it + 1);
    if (kKeys) {
      ok = ok && accumulate(L::ACC0, s_at(it), b_at(it), it, &bar.p_ready, &bar.b_empty[it % kB]);
      if (!kTwo && more) ok = ok && scores(it + 1);
    }
    ok = ok && accumulate(L::ACC1, tmem + L::DP, a_at(it), it, &bar.ds_ready, &bar.a_empty[it % kA]);
    if (more) ok = ok && dp(it + 1);
  }
  if (ok && elect_one()) umma_commit(&bar.acc_done);
  __syncwarp();
}

// What the roles of a work item share.
struct BwdItem {
  int tile, h, b;              // the 128 keys or rows that stay; a key head or a row of heads
  int i0, i1;                  // the streamed tiles: rows of the key head's rows of heads one after the other, or blocks of keys
  int key_state;               // of the keys that stay
  float mask_base;
  const uint8_t* state;        // of the batch row's blocks; null without a mask
};
template <bool kKeys>
__device__ __forceinline__ int kind_of(const CrossParams& p, const BwdItem& x, int i) {
  return kKeys ? x.key_state : x.state ? __ldg(x.state + i) : block_state_unmasked(p, i);
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

template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_loads(BwdBars& bar, const CrossParams& p, const BwdItem& x, uint32_t smem, int row_tiles, const void* f0, const void* f1, const void* a, const void* b) {
  using L = Bwd<kD>;
  constexpr int kA = L::stages_a(kKeys), kB = L::stages_b(kKeys);
  volatile int* abort_flag = &bar.abort_flag;
  if (elect_one()) {
    const int at = kKeys ? x.tile * 128 : (x.tile * 128) >> p.pack_log2;
    mbar_expect_tx(&bar.f_full, 2 * L::kTile);
    load_tile<kD>(smem + L::F0, f0, &bar.f_full, 128, at, x.h, x.b);
    load_tile<kD>(smem + L::F1, f1, &bar.f_full, 128, at, x.h, x.b);
  }
  __syncwarp();
  Ring<kA> ra;
  Ring<kB> rb;
  int as = 0, bs = 0;
  int head = kKeys ? x.h * p.per_kv + x.i0 / row_tiles : x.h / p.per_kv, row = kKeys ? x.i0 % row_tiles : 0;
  for (int i = x.i0; i < x.i1; ++i) {
    if (!kind_of<kKeys>(p, x, i)) continue;
    const int seq = kKeys ? (row * 128) >> p.pack_log2 : i * 128;
    if (!warp_ready(&bar.a_empty[ra.stage], ra.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty)) break;
    if (elect_one()) {
      mbar_expect_tx(&bar.a_full[ra.stage], L::kTile);
      load_tile<kD>(smem + L::RING + ra.stage * L::kTile, a, &bar.a_full[ra.stage], 128, seq, head, x.b);
    }
    __syncwarp();
    ++as;
    if (!warp_ready(&bar.b_empty[rb.stage], rb.parity ^ 1, abort_flag, p.status, kStatusWaitEmpty)) break;
    if (elect_one()) {
      mbar_expect_tx(&bar.b_full[rb.stage], L::kTile);
      load_tile<kD>(smem + L::RING + (kA + rb.stage) * L::kTile, b, &bar.b_full[rb.stage], 128, seq, head, x.b);
    }
    __syncwarp();
    ++bs;
    ra.next();
    rb.next();
    if (kKeys && ++row == row_tiles) {
      row = 0;
      ++head;
    }
  }
  drain(&bar.f_full, 0);
  for (int u = max(0, as - kA); u < as; ++u) drain(&bar.a_full[u % kA], (u / kA) & 1);
  for (int u = max(0, bs - kB); u < bs; ++u) drain(&bar.b_full[u % kB], (u / kB) & 1);
}

// The table of a streamed tile: {-l[128], -D[128]} of its rows, or its keys' entries.
template <int kD, bool kKeys>
__device__ __forceinline__ void bwd_tables(BwdBars& bar, const CrossParams& p, const BwdItem& x, float* tab, const float* stats, const float* D, int row_tiles, int lane) {
  Ring<Bwd<kD>::stages_a(kKeys)> ra;
  int head = kKeys ? x.h * p.per_kv + x.i0 / row_tiles : 0, row = kKeys ? x.i0 % row_tiles : 0;
  for (int i = x.i0; i < x.i1; ++i) {
    const int kind = kind_of<kKeys>(p, x, i);
    if (!kind) continue;
    float* tb = tab + ra.stage * 256;
    float2 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (kKeys) {
        const int r = row * 128 + e * 32 + lane;
        const long long at = (static_cast<long long>(x.b) * p.Hq + head) * p.R + r;
        v[e] = make_float2(-INFINITY, 0.f);
        if (r < p.R) v[e] = make_float2(-__ldg(stats + at) - (x.key_state == 2 ? x.mask_base : 0.f), -__ldcg(D + at));
      } else {
        v[e] = kind == 1 ? key_entry(p, x.b, i * 128 + e * 32 + lane, x.mask_base) : make_float2(0.f, 0.f);
      }
    }
    if (!warp_ready(&bar.a_empty[ra.stage], ra.parity ^ 1, &bar.abort_flag, p.status, kStatusWaitEmpty)) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = e * 32 + lane;
      if (kKeys) {
        tb[at] = v[e].x;
        tb[128 + at] = v[e].y;
      } else if (kind == 1) {
        reinterpret_cast<float2*>(tb)[at] = v[e];
      }
    }
    arrive_warp(&bar.tab_full[ra.stage], lane);
    ra.next();
    if (kKeys && ++row == row_tiles) {
      row = 0;
      ++head;
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

// P and dS, tile by tile; returns the number of tiles, or -1 after a wait that gave up.
template <int kD, bool kKeys>
__device__ __forceinline__ int bwd_softmax(BwdBars& bar, const CrossParams& p, const BwdItem& x, uint32_t tmem, uint32_t smem, const float* tab, const float* stats, const float* D, int warp,
                                           int lane) {
  using L = Bwd<kD>;
  constexpr bool kTwo = !kKeys || L::kTwoForKeys;
  const int w = warp >> 2, quarter = warp & 3, t = quarter * 32 + lane;
  const uint32_t at = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + w * 32;
  volatile int* abort_flag = &bar.abort_flag;
  // of the row: an entry of the mask, or statistics
  float2 entry = make_float2(0.f, 0.f);
  float neg_l = 0.f, neg_d = 0.f;
  if (kKeys) {
    if (x.key_state == 1) entry = key_entry(p, x.b, x.tile * 128 + t, x.mask_base);
  } else if (x.tile * 128 + t < p.R) {
    const long long row = (static_cast<long long>(x.b) * p.Hq + x.h) * p.R + x.tile * 128 + t;
    neg_l = -__ldg(stats + row);
    neg_d = -__ldcg(D + row);
  }
  Ring<L::stages_a(kKeys)> ra;
  Ring<kTwo ? 2 : 1> rs;
  int it = 0;
  for (int i = x.i0; i < x.i1; ++i) {
    const int kind = kind_of<kKeys>(p, x, i);
    if (!kind) continue;
    const float* tb = tab + ra.stage * 256 + (kKeys ? w * 32 : w * 64);
    const uint32_t tS = at + (rs.stage ? (kKeys ? L::S2_KEYS : L::S2_ROWS) : L::S), tDP = at + L::DP;
    if (kKeys || kind != 2)
      if (!warp_ready(&bar.tab_full[ra.stage], ra.parity, abort_flag, p.status, kStatusWaitFull)) return -1;
    if (!warp_ready(&bar.s_full[rs.stage], rs.parity, abort_flag, p.status, kStatusWaitAccum)) return -1;
    tc_fence_after_sync();
    if (kind != 2) masked_scores<kKeys>(tS, entry, reinterpret_cast<const float2*>(tb));
    uint32_t pr[32];
    make_p<kKeys>(tS, kind == 2 ? p.scale * kLog2e : 1.f, tb, kind == 2 ? neg_l - x.mask_base : neg_l, pr);
    if (kKeys) {
      tmem_st_wait();
      tc_fence_before_sync();
      arrive_warp(&bar.p_ready, lane);
    }
    if (!warp_ready(&bar.dp_full, it & 1, abort_flag, p.status, kStatusWaitAccum)) return -1;
    tc_fence_after_sync();
    if (kind != 2) {
      masked_dp<kKeys>(tDP, entry, reinterpret_cast<const float2*>(tb));
      if (!kKeys && p.mask) {        // nor of an absent key's K, which its dS of zero meets: S and dP have been read from it
        if (w == 0 && reinterpret_cast<const float2*>(tb)[t].y == -INFINITY) zero_row<kD>(smem + L::RING + ra.stage * L::kTile, 128, t);
        fence_proxy_async_smem();
      }
    }
    make_ds<kKeys>(tDP, tb + 128, neg_d, pr);
    tmem_st_wait();
    tc_fence_before_sync();
    arrive_warp(&bar.ds_ready, lane);
    ++it;
    ra.next();
    rs.next();
  }
  return it;
}

template <int kD>
__global__ void __launch_bounds__(kBwdThreads, 1)
cross_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                 const CrossParams p, const BwdOut out) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  using L = Bwd<kD>;
  static_assert(sizeof(BwdBars) <= 256, "barriers");
  BwdBars& bar = *reinterpret_cast<BwdBars*>(smem + L::BARS);
  float* tab = reinterpret_cast<float*>(smem + L::TAB);

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const bool keys = static_cast<int>(blockIdx.x) < out.key_items;
  int lin = keys ? blockIdx.x : blockIdx.x - out.key_items;
  const int parts = keys ? out.parts_k : out.parts_q, per = keys ? out.key_blocks : out.row_tiles, heads = keys ? p.Hk : p.Hq;
  const int part = lin % parts;
  lin /= parts;
  BwdItem x;
  x.tile = lin % per;
  lin /= per;
  x.h = lin % heads;
  x.b = lin / heads;
  x.state = out.state ? out.state + static_cast<long long>(x.b) * out.key_blocks : nullptr;
  const int n_all = keys ? p.per_kv * out.row_tiles : out.key_blocks, per_part = (n_all + parts - 1) / parts;
  x.i0 = part * per_part;
  x.i1 = min(n_all, x.i0 + per_part);

  if (threadIdx.x == 0) {
    mbar_init(&bar.f_full, 1);
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
    mbar_init(&bar.p_ready, kBwdSoftmaxWarps);
    mbar_init(&bar.ds_ready, kBwdSoftmaxWarps);
    mbar_init(&bar.acc_done, 1);
    bar.abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kBwdSoftmaxWarps) {
    tmem_alloc<1>(&bar.tmem_slot, 512);
    tmem_relinquish<1>();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = bar.tmem_slot;
  pdl_entry();
  const uint32_t base = smem_u32(smem);
  x.key_state = !keys ? 0 : x.state ? __ldg(x.state + x.tile) : block_state_unmasked(p, x.tile);
  x.mask_base = p.base ? __ldg(p.base + x.b) : 0.f;
  if (keys && x.key_state == 0) x.i1 = x.i0;                // no key of the block takes part

  if (warp == kBwdSoftmaxWarps + 1) {
    if (keys) bwd_loads<kD, true>(bar, p, x, base, out.row_tiles, &tmK, &tmV, &tmQ, &tmDO);
    else bwd_loads<kD, false>(bar, p, x, base, out.row_tiles, &tmQ, &tmDO, &tmK, &tmV);
  } else if (warp == kBwdSoftmaxWarps + 2) {
    if (keys) bwd_tables<kD, true>(bar, p, x, tab, out.stats, out.D, out.row_tiles, lane);
    else bwd_tables<kD, false>(bar, p, x, tab, out.stats, out.D, out.row_tiles, lane);
  } else if (warp == kBwdSoftmaxWarps) {
    int n = x.i1 - x.i0;
    if (keys) {
      bwd_products<kD, true>(bar, p.status, tmem, base, n);
    } else {
      for (int i = x.i0; i < x.i1; ++i) n -= kind_of<false>(p, x, i) == 0;
      bwd_products<kD, false>(bar, p.status, tmem, base, n);
    }
  } else {
    const int n = keys ? bwd_softmax<kD, true>(bar, p, x, tmem, base, tab, out.stats, out.D, warp, lane) : bwd_softmax<kD, false>(bar, p, x, tmem, base, tab, out.stats, out.D, warp, lane);
    if (n == 0 || (n > 0 && warp_ready(&bar.acc_done, 0, &bar.abort_flag, p.status, kStatusWaitAccum))) {
      tc_fence_after_sync();
      // keys: half of the warps write dK, the others dV; rows: all of them dQ
      const int w = warp >> 2, quarter = warp & 3, r = x.tile * 128 + quarter * 32 + lane;
      const bool inside = keys ? r < p.Sk : r < p.R, is_v = keys && w >= 2;
      const int step = keys ? kD / 2 : kD / 4, c0 = (keys ? w & 1 : w) * step, c1 = c0 + step;
      const uint32_t acc = tmem + (is_v ? L::ACC0 : L::ACC1) + (static_cast<uint32_t>(quarter * 32) << 16);
      const float mul = is_v ? 1.f : p.scale;
      const long long line = keys ? (static_cast<long long>(x.b) * p.Hk + x.h) * p.Sk + r : (static_cast<long long>(x.b) * p.Hq + x.h) * p.R + r;
      const long long lines = keys ? static_cast<long long>(p.B) * p.Hk * p.Sk : static_cast<long long>(p.B) * p.Hq * p.R;
      float* part_at = nullptr;
      __nv_bfloat16* at = nullptr;
      if (parts > 1) part_at = (keys ? (is_v ? out.part_v : out.part_k) : out.part_q) + (part * lines + line) * kD;
      else if (keys) at = (is_v ? out.dv : out.dk) + x.b * out.ksb + r * out.kss + x.h * out.ksh;
      else at = out_row(p, out.dq, out.qsb, out.qss, out.qsh, x.b, x.h, r);
#pragma unroll 1
      for (int c = c0; c < c1; c += 16) {
        uint32_t v[16];
        if (n > 0) {
          tmem_ld16(acc + c, v);
          tmem_ld_wait();
        }
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (n > 0) asm volatile("" : "+r"(v[e]));
          f[e] = n > 0 ? __uint_as_float(v[e]) * mul : 0.f;
        }
        if (inside) {
          if (parts > 1) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(part_at + c + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 8) *reinterpret_cast<uint4*>(at + c + e) = pack8(f + e);
          }
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

// Before: D = rowsum(dO o), eight values a lane; and, in the blocks behind, what the mask says of each block of keys.
template <int kD>
__global__ void __launch_bounds__(256) cross_pre_kernel(const CrossParams p, const __nv_bfloat16* __restrict__ o, const long long osb, const long long oss, const long long osh,
                                                        const __nv_bfloat16* __restrict__ d_o, const long long gsb, const long long gss, const long long gsh,
                                                        float* __restrict__ D, uint8_t* __restrict__ state, const int row_blocks) {
  pdl_entry();
  const int lane = threadIdx.x & 31;
  if (static_cast<int>(blockIdx.x) >= row_blocks) {
    const int nblk = (p.Sk + kKeys - 1) / kKeys;
    const long long at = (blockIdx.x - row_blocks) * 8ll + (threadIdx.x >> 5);
    if (at >= static_cast<long long>(p.B) * nblk) return;
    const int s = block_state(p, static_cast<int>(at / nblk), static_cast<int>(at % nblk), lane);
    if (lane == 0) state[at] = static_cast<uint8_t>(s);
    return;
  }
  constexpr int kLanes = kD / 8;
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.R;
  const int c = (threadIdx.x % kLanes) * 8;
  const unsigned m = kLanes == 16 ? 0xffffu << (lane & 16) : 0xffu << (lane & 24);
  for (long long row = (blockIdx.x * 256ll + threadIdx.x) / kLanes; row < rows; row += row_blocks * 256ll / kLanes) {
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

// After: parts added in their order, rounded to bf16. Rows of [B, heads, n] (rows of heads, or key heads), four values a lane.
template <int kD>
__global__ void __launch_bounds__(256) cross_sum_kernel(const CrossParams p, const BwdOut out) {
  pdl_entry();
  constexpr int kLanes = kD / 4;
  const long long q_rows = out.parts_q > 1 ? static_cast<long long>(p.B) * p.Hq * p.R : 0, k_rows = out.parts_k > 1 ? static_cast<long long>(p.B) * p.Hk * p.Sk : 0;
  const int c = (threadIdx.x % kLanes) * 4;
  for (long long row = (blockIdx.x * 256ll + threadIdx.x) / kLanes; row < q_rows + 2 * k_rows; row += gridDim.x * 256ll / kLanes) {
    const bool q = row < q_rows, v = !q && row >= q_rows + k_rows;
    const long long at = q ? row : row - q_rows - (v ? k_rows : 0), rows = q ? q_rows : k_rows;
    const float* src = (q ? out.part_q : v ? out.part_v : out.part_k) + at * kD + c;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < (q ? out.parts_q : out.parts_k); ++i) {
      const float4 x = *reinterpret_cast<const float4*>(src + i * rows * kD);
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    __nv_bfloat16* dst;
    if (q) {
      const long long bh = at / p.R;
      dst = out_row(p, out.dq, out.qsb, out.qss, out.qsh, static_cast<int>(bh / p.Hq), static_cast<int>(bh % p.Hq), static_cast<int>(at % p.R));
    } else {
      const long long bh = at / p.Sk;
      dst = (v ? out.dv : out.dk) + (bh / p.Hk) * out.ksb + (at % p.Sk) * out.kss + (bh % p.Hk) * out.ksh;
    }
    *reinterpret_cast<uint2*>(dst + c) = make_uint2(pack2(acc.x, acc.y), pack2(acc.z, acc.w));
  }
}

// ------------------------------------------------------------------------------------------ host
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
  p.mask = a.mask;
  p.mask_stride = a.mask_stride;
  p.mask_bool = a.mask_bool;
  p.base = a.mask && !a.mask_bool && a.stats ? a.stats + static_cast<long long>(a.B) * a.H * a.Sq : nullptr;
  p.scale = a.scale;
  p.table = !(a.scale > 0.f);
  p.status = a.status;
  return true;
}

int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Parts of the keys in the forward pass: where the tiles leave CTA slots (two an SM) empty, as many as fill them, of two blocks at least. Each costs a tile of fp32 sums
// to memory and back.
int fwd_parts(const CrossParams& p) {
  const long long tiles = static_cast<long long>(ceil_div(p.R, 128)) * p.Hq * p.B, slots = 2ll * sm_count();
  const int nblk = ceil_div(p.Sk, kKeys);
  long long parts = 1;
  if (tiles * 2 <= slots) parts = slots / tiles;
  if (parts > nblk / 2) parts = nblk / 2;
  if (parts < 1) parts = 1;
  const int least = ceil_div(nblk, kMaxBlocks);
  if (parts < least) parts = least;
  return ceil_div(nblk, ceil_div(nblk, parts));
}

// Parts of an item's streamed tiles in the backward pass: an item longer than its share of all the work holds up the launch's end.
void bwd_parts(const CrossParams& p, int& parts_q, int& parts_k) {
  const long long n_q = ceil_div(p.Sk, 128), n_k = static_cast<long long>(p.per_kv) * ceil_div(p.R, 128);
  const long long items_q = static_cast<long long>(ceil_div(p.R, 128)) * p.Hq * p.B, items_k = static_cast<long long>(ceil_div(p.Sk, 128)) * p.Hk * p.B;
  const long long share = (n_q * items_q + n_k * items_k) / sm_count();
  const long long least = share > 4 ? share : 4;
  parts_q = n_q > least ? ceil_div(n_q, least) : 1;
  parts_k = n_k > least ? ceil_div(n_k, least) : 1;
  parts_q = ceil_div(n_q, ceil_div(n_q, parts_q));
  parts_k = ceil_div(n_k, ceil_div(n_k, parts_k));
}

template <int kD>
int cross_fwd(const fb_cross_args& a, const CrossParams& p, int pack, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  int e = make_tmap_rows(&tq, a.q, kD, pack, a.Sq, p.Hq, a.B, a.q_strides[0], a.q_strides[1], a.q_strides[2]);
  if (!e) e = make_tmap_rows(&tk, a.k, kD, 1, a.Sk, a.Hk, a.B, a.k_strides[0], a.k_strides[1], a.k_strides[2]);
  if (!e) e = make_tmap_rows(&tv, a.v, kD, 1, a.Sk, a.Hk, a.B, a.v_strides[0], a.v_strides[1], a.v_strides[2]);
  if (e) return e;
  FwdOut out = {};
  out.o = static_cast<__nv_bfloat16*>(a.o);
  out.osb = a.o_strides[0];
  out.oss = a.o_strides[1];
  out.osh = a.o_strides[2];
  out.stats = a.stats;
  out.parts = fwd_parts(p);
  out.blocks_per_part = ceil_div(ceil_div(p.Sk, kKeys), out.parts);
  out.n_tiles = ceil_div(p.R, 128);
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.R;
  if (out.parts > 1) {
    if (!a.workspace) return -3;
    out.part_ml = reinterpret_cast<float2*>(a.workspace);
    out.part_o = a.workspace + (out.parts * rows * 2 + 3) / 4 * 4;
  }
  const long long ctas = static_cast<long long>(out.n_tiles) * p.Hq * p.B * out.parts;
  if (ctas > 0x7fffffffll) return -4;
  const int smem = Fwd<kD>::bytes(out.blocks_per_part);
  if (const cudaError_t err = allow_smem<cross_fwd_kernel<kD>>(Fwd<kD>::bytes(kMaxBlocks), true)) return static_cast<int>(err);
  if (const cudaError_t err = launch_pdl(cross_fwd_kernel<kD>, dim3(static_cast<unsigned>(ctas)), dim3(kFwdThreads), static_cast<size_t>(smem), stream, tq, tk, tv, p, out))
    return static_cast<int>(err);
  if (out.parts > 1) {
    const long long blocks = (rows * (kD / 4) + 255) / 256;
    launch_pdl(cross_join_kernel<kD>, dim3(static_cast<unsigned>(blocks < 16ll * sm_count() ? blocks : 16ll * sm_count())), dim3(256), 0, stream, p, out);
  }
  return static_cast<int>(cudaGetLastError());
}

// Floats of the backward pass's workspace: D, the parts' sums, and bytes of block states.
struct BwdSpace {
  long long D, state, part_q, part_k, part_v, total;
};
BwdSpace bwd_space(const CrossParams& p, int D, int parts_q, int parts_k) {
  const auto round = [](long long n) { return (n + 31) / 32 * 32; };
  const long long q_rows = static_cast<long long>(p.B) * p.Hq * p.R, k_rows = static_cast<long long>(p.B) * p.Hk * p.Sk;
  BwdSpace s;
  s.D = 0;
  s.state = round(q_rows);
  s.part_q = s.state + (p.mask ? round((static_cast<long long>(p.B) * ceil_div(p.Sk, kKeys) + 3) / 4) : 0);
  s.part_k = s.part_q + (parts_q > 1 ? parts_q * q_rows * D : 0);
  s.part_v = s.part_k + (parts_k > 1 ? parts_k * k_rows * D : 0);
  s.total = s.part_v + (parts_k > 1 ? parts_k * k_rows * D : 0);
  return s;
}

template <int kD>
int cross_bwd(const fb_cross_args& a, const CrossParams& p, int pack, cudaStream_t stream) {
  CUtensorMap tq, tk, tv, tdo;
  int e = make_tmap_rows(&tq, a.q, kD, pack, a.Sq, p.Hq, a.B, a.q_strides[0], a.q_strides[1], a.q_strides[2]);
  if (!e) e = make_tmap_rows(&tk, a.k, kD, 1, a.Sk, a.Hk, a.B, a.k_strides[0], a.k_strides[1], a.k_strides[2]);
  if (!e) e = make_tmap_rows(&tv, a.v, kD, 1, a.Sk, a.Hk, a.B, a.v_strides[0], a.v_strides[1], a.v_strides[2]);
  if (!e) e = make_tmap_rows(&tdo, a.d_o, kD, pack, a.Sq, p.Hq, a.B, a.do_strides[0], a.do_strides[1], a.do_strides[2]);
  if (e) return e;
  BwdOut out = {};
  bwd_parts(p, out.parts_q, out.parts_k);
  const BwdSpace space = bwd_space(p, kD, out.parts_q, out.parts_k);
  if (!a.workspace || !a.stats) return -3;
  float* D = a.workspace + space.D;
  uint8_t* state = p.mask ? reinterpret_cast<uint8_t*>(a.workspace + space.state) : nullptr;
  out.stats = a.stats;
  out.D = D;
  out.state = state;
  out.part_q = a.workspace + space.part_q;
  out.part_k = a.workspace + space.part_k;
  out.part_v = a.workspace + space.part_v;
  out.dq = static_cast<__nv_bfloat16*>(a.dq);
  out.dk = static_cast<__nv_bfloat16*>(a.dk);
  out.dv = static_cast<__nv_bfloat16*>(a.dv);
  out.qsb = a.dq_strides[0]; out.qss = a.dq_strides[1]; out.qsh = a.dq_strides[2];
  out.ksb = a.dk_strides[0]; out.kss = a.dk_strides[1]; out.ksh = a.dk_strides[2];
  out.row_tiles = ceil_div(p.R, 128);
  out.key_blocks = ceil_div(p.Sk, 128);
  const long long rows = static_cast<long long>(p.B) * p.Hq * p.R;
  const long long key_items = static_cast<long long>(out.key_blocks) * p.Hk * p.B * out.parts_k, items = key_items + static_cast<long long>(out.row_tiles) * p.Hq * p.B * out.parts_q;
  if (items > 0x7fffffffll) return -4;
  out.key_items = static_cast<int>(key_items);
  const long long want = (rows * (kD / 8) + 255) / 256;
  const int row_blocks = static_cast<int>(want < 16ll * sm_count() ? want : 16ll * sm_count());
  const long long state_blocks = state ? (static_cast<long long>(p.B) * out.key_blocks + 7) / 8 : 0;
  if (state_blocks > 0x3fffffffll) return -4;
  launch_pdl(cross_pre_kernel<kD>, dim3(row_blocks + static_cast<unsigned>(state_blocks)), dim3(256), 0, stream, p, static_cast<const __nv_bfloat16*>(a.o), a.o_strides[0], a.o_strides[1],
             a.o_strides[2], static_cast<const __nv_bfloat16*>(a.d_o), a.do_strides[0], a.do_strides[1], a.do_strides[2], D, state, row_blocks);
  constexpr int smem = Bwd<kD>::TOTAL + 1024;
  if (const cudaError_t err = allow_smem<cross_bwd_kernel<kD>>(smem)) return static_cast<int>(err);
  if (const cudaError_t err = launch_pdl(cross_bwd_kernel<kD>, dim3(static_cast<unsigned>(items)), dim3(kBwdThreads), static_cast<size_t>(smem), stream, tq, tk, tv, tdo,
                                         p, out))
    return static_cast<int>(err);
  if (out.parts_q > 1 || out.parts_k > 1) {
    const long long sum_rows = (out.parts_q > 1 ? rows : 0) + (out.parts_k > 1 ? 2ll * p.B * p.Hk * p.Sk : 0), blocks = (sum_rows * (kD / 4) + 255) / 256;
    launch_pdl(cross_sum_kernel<kD>, dim3(static_cast<unsigned>(blocks < 16ll * sm_count() ? blocks : 16ll * sm_count())), dim3(256), 0, stream, p, out);
  }
  return static_cast<int>(cudaGetLastError());
}

bool rows_ok(const void* p, const long long* st) { return strides_ok(p, st[0], st[1], st[2]); }

}  // namespace
}  // namespace fb

extern "C" long long fb_cross_workspace(const fb_cross_args* args, int backward) {
  using namespace fb;
  CrossParams p = {};
  int pack;
  if (!make_cross(*args, p, pack)) return -4;
  if (backward) {
    int parts_q, parts_k;
    bwd_parts(p, parts_q, parts_k);
    return bwd_space(p, args->D, parts_q, parts_k).total;
  }
  const long long parts = fwd_parts(p), rows = static_cast<long long>(p.B) * p.Hq * p.R;
  return parts > 1 ? (parts * rows * 2 + 3) / 4 * 4 + parts * rows * args->D : 0;
}

extern "C" int fb_cross_attn_fwd(const fb_cross_args* args, void* stream) {
  using namespace fb;
  const fb_cross_args& a = *args;
  CrossParams p = {};
  int pack;
  if (!make_cross(a, p, pack)) return -4;
  if (!rows_ok(a.q, a.q_strides) || !rows_ok(a.k, a.k_strides) || !rows_ok(a.v, a.v_strides) || !rows_ok(a.o, a.o_strides)) return -3;
  const auto s = static_cast<cudaStream_t>(stream);
  return a.D == 64 ? cross_fwd<64>(a, p, pack, s) : cross_fwd<128>(a, p, pack, s);
}

extern "C" int fb_cross_attn_bwd(const fb_cross_args* args, void* stream) {
  using namespace fb;
  const fb_cross_args& a = *args;
  CrossParams p = {};
  int pack;
  if (!make_cross(a, p, pack)) return -4;
  if (!rows_ok(a.q, a.q_strides) || !rows_ok(a.k, a.k_strides) || !rows_ok(a.v, a.v_strides) || !rows_ok(a.o, a.o_strides) || !rows_ok(a.d_o, a.do_strides) ||
      !rows_ok(a.dq, a.dq_strides) || !rows_ok(a.dk, a.dk_strides) || !rows_ok(a.dv, a.dk_strides))
    return -3;
  const auto s = static_cast<cudaStream_t>(stream);
  return a.D == 64 ? cross_bwd<64>(a, p, pack, s) : cross_bwd<128>(a, p, pack, s);
}
