// Attention of new tokens over a KV cache that already holds their K and V (flb_extend_fwd): chunked
// prefill, speculative tokens, batches that mix chunks and single tokens, and single-token decode
// over an 8-bit cache. 16-bit or int8 caches, contiguous or paged, ragged sequences.
//
// The mathematics. Row i of a sequence with L keys and n rows sees keys j < L - n + i + 1 (causal)
// or j < L: o_i = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - M), s_j = scale log2(e) q_i . k_j
// and M any reference point near the row's maximum. An int8 cache holds k_j = sk_j K_j and
// v_j = sv_j V_j with integers K, V of at most 127: both integers are exact in bf16 and fp16, the scale
// of K multiplies a column of S, and the scale of V joins the exponent,
//     w_j = 2^(z_j - M),  z_j = s_j + log2 sv_j,  o = sum_j w_j V_j / sum_j (w_j / sv_j),
// so the weights that enter the second product as fp16 lie in (0, 2^8] whatever the size of the
// scales. Weights below 2^-25 are 0 there (N of them make o differ by less than N 2^-18 steps of the row
// with the largest weight); the sum of w_j / sv_j in fp32 keeps them.
//
// What bounds it. An item of 2 x 128 rows reads its K/V bytes once, so few rows per sequence are bound
// by HBM (2 H_kv D bytes per key at 8 bits, twice that at 16) and chunks of hundreds of rows by the
// tensor cores and the exponentials. (Items of the same keys run at different times, and L2 serves little
// of that: 4 x 512 rows after 16K keys, 8 items per KV head, read 2.1 GB for 277 MB of K and V.) Measured on
// B200 as device time of a graph of two calls: 2048 rows after 16K bf16 keys (H 32, H_kv 8, D 128) 479 us,
// 1.22 PFLOP/s (calls one after the other run at the power limit: 546-560 us, 1.04-1.07 PFLOP/s); one
// row of 8 sequences of 24K bf16 keys (806 MB) 129 us, 6.3 TB/s; prompts of 4 x 2500-4095 rows
// (fp16, 16 heads, D 64) 151 us, 0.56 PFLOP/s; 2 x 512 rows after 16K int8 keys (D 128) 467 us, 0.60
// PFLOP/s (its softmax takes 5000 clocks per tile where that of 16 bits takes 1800).
//
// Roundings to fewer than 32 bits: the weights, to the type of the V operand of tcgen05.mma, which is the
// cache's at 16 bits (bf16 2^-8, fp16 2^-11) and fp16 for codes; and the result, to q's type. Over bf16
// caches that is 0.0021-0.0023 of the result's norm against 0.0016 with fp32 weights. Scores, reference
// points, sums, O and the partials are fp32. log2 of a V scale is lg2.approx, off by at most 2^-22 of
// itself.
//
// How it is split.
//  * A tile of 128 score rows is (tokens x the query heads of one KV head): head h of token i is
//    row i * group + h, so K/V are read once per group and a few tokens fill a tile. Q comes by
//    TMA as a [64 columns x group x tokens] box.
//  * An item is two such tiles of one (sequence, KV head), one softmax warpgroup each, over the keys
//    its last row sees. When its tokens fit in one tile, both warpgroups work on that tile, on
//    alternate key tiles (a chain of Q K^T, softmax, P V is latency bound: two of them per SM are
//    twice the rate), and the first joins the two results through TMEM at the end.
//  * The steps of both chains take the S buffers in TMEM in turn. Two fit beside O at head_dim 128; at
//    64 there is a third, so a chain finds its next scores ready: 169 -> 146 us for the prompts above.
//  * One CTA per SM. The items' key tiles, in the order (KV head, sequence, item, key tile), are cut
//    into equal shares (a tile of a two-tile item counts twice, and each item has a fixed part), so
//    a long cache with few rows spreads over all SMs and ragged batches stay balanced. Every CTA
//    finds its share from cu_seqlens and seq_lens on the device. An item that is cut leaves fp32
//    partials (at most two per CTA) that extend_merge_kernel joins in key order.
//  * Warps: two softmax warpgroups, a TMA producer, the MMA issuer, and for int8 a warpgroup each for
//    K and V that turns [128 x D] code tiles into the 16-bit tiles the tensor cores read.
//  * Keys past a sequence's length are masked in S and their V rows are zeroed in shared memory
//    (cache rows past the length may hold anything, and 0 * NaN is NaN).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "extend_work.cuh"

namespace flb {
namespace {

constexpr int kBM = 128;              // score rows per tile
constexpr int kBoxBytes = kBM * 128;  // a swizzled [128 rows x 64 columns] 16-bit box
constexpr uint32_t kTmemCols = 512;   // the S buffers | O0 | O1

constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kConvertWarp = 12;      // int8: warps 12-15 (K and scales), 16-19 (V)

// 16-bit: 128 KB of K/V tiles beside the two Q tiles. int8: 96 KB of 16-bit tiles, 48 KB of codes
// (what is in flight from HBM). K and V have rings of their own, and K runs one tile ahead of V:
// with 96 KB in one ring the next K tile waited for the last P V, and the MMA warp with it, which
// put both chains in line (8 sequences of 24K int8 keys, one row: 297 us).
template <int D, bool kInt8>
struct Geometry {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  static constexpr int kBoxes = D / 64;
  // S buffers of 128 TMEM columns that the steps of both chains take in turn: what O leaves.
  static constexpr int kSBufs = D == 64 ? 3 : 2;
  static constexpr uint32_t kOCol = kSBufs * 128;        // O of chain 0; chain 1's follows
  static_assert(kOCol + 2 * D <= kTmemCols, "S and O fit in TMEM");
  static constexpr int kTileBytes = kBM * D * 2;
  static constexpr int kCodeBytes = kBN * D;
  static constexpr int kKSlots = 2 * (128 / D);
  static constexpr int kVSlots = (kInt8 ? 1 : 2) * (128 / D);
  static constexpr int kSlots = kKSlots + kVSlots;
  static constexpr int kCodeSlots = kInt8 ? 3 * (128 / D) : 0;
  // Key tiles whose scales are held: a K tile is converted once Q K^T of the tile kKSlots earlier
  // has been issued, which follows the softmax of tiles kSBufs or more before that one.
  static constexpr int kScaleSlots = kInt8 ? kKSlots + kSBufs : 0;
  // mult, log2 sv and 1 / sv of each key; then, from each warp of 32 keys, a byte: whether the row sum
  // needs care (softmax_tile_int8).
  static constexpr int kCareAt = 3 * kBN;
  static constexpr int kScaleWords = kCareAt + 4;
  static constexpr int kScaleBytes = kScaleSlots * kScaleWords * 4;
  static constexpr int kRingOffset = 2 * kTileBytes;
  static constexpr int kCodeOffset = kRingOffset + kSlots * kTileBytes;
  static constexpr int kScaleOffset = kCodeOffset + kCodeSlots * kCodeBytes;
  static constexpr int kTailOffset = kScaleOffset + kScaleBytes;
  static constexpr int kThreads = kInt8 ? 640 : 384;
  // The register split (setmaxnreg) must not exceed what the CTA is launched with.
  static constexpr int kLaunchRegs = kInt8 ? 96 : 168;
  static constexpr int kSoftmaxRegs = kInt8 ? 128 : 216;
  static constexpr int kOtherRegs = 72;
  static_assert(2 * 128 * kSoftmaxRegs + (kThreads - 256) * kOtherRegs <= kThreads * kLaunchRegs,
                "the register split must fit in the launch's registers");
  static_assert(kMaxBatch * 4 <= kSlots * kTileBytes, "prefix sums fit in the rings");
};

template <int kKSlots, int kVSlots, int kCodeSlots, int kScaleSlots, int kSBufs>
struct Shared {
  uint64_t q_full[2];
  uint64_t q_free[2];        // the last Q K^T of an item that reads a Q tile has completed
  uint64_t k_full[kKSlots];
  uint64_t k_empty[kKSlots];
  uint64_t v_full[kVSlots];
  uint64_t v_empty[kVSlots];
  uint64_t code_full[kCodeSlots + 1];
  uint64_t code_empty[kCodeSlots + 1];
  uint64_t scale_full[kScaleSlots + 1];
  uint64_t s_full[kSBufs];
  uint64_t p_half[kSBufs][2];   // P of keys 0-63 / 64-127 of a tile stored in TMEM
  uint64_t o_full[2];
  uint64_t x_ready, x_done;  // the chains' meeting at the end of a joined segment
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
  Share share;
  float2 x_ml[kBM];          // (m, l) of the second chain's rows
};

// --------------------------------------------------------------------------------------------
// Operand descriptors (see prefill.cu: any tile and k-step is one add to a base descriptor)
// --------------------------------------------------------------------------------------------

struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ explicit Desc(uint64_t d)
      : lo(static_cast<uint32_t>(d)), hi(static_cast<uint32_t>(d >> 32)) {}
  __device__ __forceinline__ Desc(uint32_t l, uint32_t h) : lo(l), hi(h) {}
  __device__ __forceinline__ Desc at(uint32_t bytes) const { return Desc(lo + (bytes >> 4), hi); }
  __device__ __forceinline__ uint64_t u64() const {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
  }
};
constexpr uint32_t kmajor_step(int kk) { return (kk >> 2) * kBoxBytes + (kk & 3) * 32; }
constexpr uint32_t mnmajor_step(int kk) { return kk * 2048; }

// Whether the phase with the given parity has completed, without waiting.
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// --------------------------------------------------------------------------------------------
// 8-bit codes
// --------------------------------------------------------------------------------------------

// A [128 x D] code tile to a 16-bit tile of 128-byte-swizzled [128 x 64] boxes, by 128 threads:
// 16 codes each per step. The lanes of columns 64-127 store their two chunks in the other order,
// which keeps the eight lanes of a store phase on different banks.
template <typename T, int D>
__device__ __forceinline__ void convert_tile(const uint8_t* codes, uint8_t* tile, int tid) {
  constexpr int kChunks = D / 16;
  constexpr int kBatch = 4;   // loads in flight: the compiler cannot move one past a store
  const int c = tid % kChunks, swap = c >> 2;
  const int row0 = tid / kChunks;
  uint8_t* box = tile + (c >> 2) * kBoxBytes;
#pragma unroll 1
  for (int i0 = 0; i0 < kChunks; i0 += kBatch) {
    uint4 x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      x[i] = *reinterpret_cast<const uint4*>(codes + ((i0 + i) * 128 + tid) * 16);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      uint4 y0, y1;
      codes_to_16bit<T>(x[i].x, y0.x, y0.y);
      codes_to_16bit<T>(x[i].y, y0.z, y0.w);
      codes_to_16bit<T>(x[i].z, y1.x, y1.y);
      codes_to_16bit<T>(x[i].w, y1.z, y1.w);
      const int row = row0 + (i0 + i) * (128 / kChunks), chunk = (2 * c) & 7;
      *reinterpret_cast<uint4*>(box + sw128_offset(row, chunk + swap)) = swap ? y1 : y0;
      *reinterpret_cast<uint4*>(box + sw128_offset(row, chunk + 1 - swap)) = swap ? y0 : y1;
    }
  }
}

// --------------------------------------------------------------------------------------------
// Softmax
// --------------------------------------------------------------------------------------------

// The barrier phase by which P V of a chain's previous step has completed: the release of its V tile
// (in a two-tile item by chain 1's P V, which does not wait for this step of either chain). `needed`
// when this step's scores do not say so, that is when fewer than kSBufs steps lie between: only then
// is the phase sure to be the barrier's current or last one, whatever the number of V slots.
struct PrevPv {
  uint64_t* bar;
  uint32_t parity;
  bool needed;
};

// The reference point of a row moves only when its maximum mt (log2 domain) passes it by more than
// 2^8; the row sum and O (in TMEM) follow, once P V of the chain's previous step has completed.
// This step's waits for the first half of P.
template <int D>
__device__ __forceinline__ void move_reference(float mt, float& m_ref, float& l_sum,
                                               uint32_t taddr_o, const PrevPv& prev,
                                               const WaitGuard& guard) {
  float m_new = m_ref;
  if (m_ref == -INFINITY || mt > m_ref + kRescaleThreshold) m_new = fmaxf(m_ref, mt);
  const bool rescale = (m_new != m_ref) && (m_ref != -INFINITY);
  const float factor = rescale ? ex2(m_ref - m_new) : 1.f;
  if (rescale) l_sum = scale_sum(l_sum, m_ref - m_new);
  m_ref = m_new;
  if (__any_sync(0xffffffffu, rescale)) {
    if (prev.needed) {
      if (!mbar_wait(prev.bar, prev.parity, guard)) return;   // the next wait gives up as well
      tc_fence_after();
    }
#pragma unroll 1
    for (int i = 0; i < D / 16; ++i) {
      uint32_t ov[16];
      tmem_ld16(taddr_o + i * 16, ov);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * factor);
      tmem_st16(taddr_o + i * 16, ov);
    }
  }
}

// Publishes one half of P (64 keys) to the MMA warp.
__device__ __forceinline__ void publish_half(uint64_t* bar) {
  tmem_st_wait();
  tc_fence_before();
  mbar_arrive(bar);
}

// One key tile of one score row of a 16-bit cache: scores in 128 TMEM columns, keys at or past
// `visible` hidden when `masked`; P as packed pairs over the first 64 columns.
template <typename T, int D>
__device__ __forceinline__ void softmax_tile(uint32_t taddr_s, uint32_t taddr_o, float sl2,
                                             bool masked, int visible, float& m_ref, float& l_sum,
                                             uint64_t* bars, const PrevPv& prev,
                                             const WaitGuard& guard) {
  uint32_t sr[128];
#pragma unroll
  for (int i = 0; i < 128; i += 32)
    tmem_ld32(taddr_s + i, *reinterpret_cast<uint32_t(*)[32]>(&sr[i]));
  tmem_ld_wait();
  float* sf = reinterpret_cast<float*>(sr);
  if (masked) {
#pragma unroll
    for (int i = 0; i < 128; ++i) {
      if (i >= visible) sf[i] = -INFINITY;
    }
  }
  float mx8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mx8[i] = fmaxf(sf[i], sf[i + 8]);
#pragma unroll
  for (int i0 = 16; i0 < 128; i0 += 16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) mx8[i] = fmax3(mx8[i], sf[i0 + 2 * i], sf[i0 + 2 * i + 1]);
  }
  const float mx = fmaxf(fmax3(mx8[0], mx8[1], mx8[2]),
                         fmaxf(fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
  move_reference<D>(mx == -INFINITY ? -INFINITY : mx * sl2, m_ref, l_sum, taddr_o, prev,
                    guard);
  const float nref = m_ref == -INFINITY ? 0.f : -m_ref;
  float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t pk[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const int i = half * 64 + 2 * c, acc = (c & 1) * 2;
      float x0, x1;
      ffma2(x0, x1, sf[i], sf[i + 1], sl2, sl2, nref, nref);
      const float p0 = ex2(x0), p1 = ex2(x1);
      fadd2(ps[acc], ps[acc + 1], ps[acc], ps[acc + 1], p0, p1);
      pk[c] = pack2<T>(p0, p1);
    }
    tmem_st32(taddr_s + half * 32, pk);
    publish_half(&bars[half]);
  }
  l_sum += (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

// The second pass over an int8 tile: weights from the scaled scores z in TMEM, and their sum over
// w / sv. kWide: the sum's terms 2^(z - log2 sv - M) by exponentials of their own.
template <bool kWide>
__device__ __forceinline__ void weights_int8(uint32_t taddr_s, const float* scales, float nref,
                                             float (&ps)[4], uint64_t* bars) {
  constexpr int kCols = kWide ? 16 : 32;   // the rare form must not cost the usual one registers
#pragma unroll 1
  for (int c0 = 0; c0 < 128; c0 += kCols) {
    uint32_t zr[kCols], pk[kCols / 2];
    if constexpr (kWide) tmem_ld16(taddr_s + c0, zr);
    else tmem_ld32(taddr_s + c0, zr);
    tmem_ld_wait();
    float* z = reinterpret_cast<float*>(zr);
#pragma unroll
    for (int i = 0; i < kCols; i += 4) {
      const float4 by = *reinterpret_cast<const float4*>(scales + (kWide ? 1 : 2) * kBN + c0 + i);
      float p[4];
      fadd2(p[0], p[1], z[i], z[i + 1], nref, nref);
      fadd2(p[2], p[3], z[i + 2], z[i + 3], nref, nref);
      if constexpr (kWide) {
        const float r[4] = {by.x, by.y, by.z, by.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // The square of a root: the term may be below the exponential's range, 2^-126. Keys past
          // the length: log2 sv is -inf.
          const float root = ex2(0.5f * (p[e] - r[e]));
          ps[e] = r[e] == -INFINITY ? ps[e] : fmaf(root, root, ps[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = ex2(p[e]);
      if constexpr (!kWide) {
        ffma2(ps[0], ps[1], p[0], p[1], by.x, by.y, ps[0], ps[1]);
        ffma2(ps[2], ps[3], p[2], p[3], by.z, by.w, ps[2], ps[3]);
      }
      pk[i / 2] = pack2<__half>(p[0], p[1]);
      pk[i / 2 + 1] = pack2<__half>(p[2], p[3]);
    }
    if constexpr (kWide) tmem_st8(taddr_s + c0 / 2, pk);
    else tmem_st16(taddr_s + c0 / 2, pk);
    if (((c0 + kCols) & 63) == 0) publish_half(&bars[c0 / 64]);
  }
}

// The same over an int8 cache, with fp16 weights. `scales` holds the tile's per-key numbers in shared
// memory: mult, log2 sv and 1 / sv. They are read once: the scaled scores z go back to TMEM between the
// two passes. 32 columns at a time leave registers to read ahead; with all 128 in registers the
// loop spilled, and the spills cost more than the softmax.
//
// A weight under 2^-126 is 0, and its term w / sv with it, however small sv is: a row of zeros in V has
// sv = 2^-100. What a tile can lose that way is 128 terms under 2^-126 / sv. With scales in [2^-40, 2^45] so
// far in the segment that is below 2^-34 of the row's sum, since a row that sees a key has a sum of at least
// 1 / sv of one of them. With others it is below 2^-19, which over all tiles of the segment stays below 2^-20
// of a sum of at least `need`, twice their number. Else the terms take exponentials of their own.
template <int D>
__device__ __forceinline__ void softmax_tile_int8(uint32_t taddr_s, uint32_t taddr_o,
                                                  const float* scales, float need, bool masked,
                                                  int visible, float& m_ref, float& l_sum, uint64_t* bars,
                                                  const PrevPv& prev, const WaitGuard& guard) {
  float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
  for (int c0 = 0; c0 < 128; c0 += 32) {
    uint32_t sr[32];
    tmem_ld32(taddr_s + c0, sr);
    tmem_ld_wait();
    float* z = reinterpret_cast<float*>(sr);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 mul = *reinterpret_cast<const float4*>(scales + c0 + i);
      const float4 add = *reinterpret_cast<const float4*>(scales + kBN + c0 + i);
      ffma2(z[i], z[i + 1], z[i], z[i + 1], mul.x, mul.y, add.x, add.y);
      ffma2(z[i + 2], z[i + 3], z[i + 2], z[i + 3], mul.z, mul.w, add.z, add.w);
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (c0 + i >= visible) z[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mx4[e] = fmax3(mx4[e], z[i + 2 * e], z[i + 2 * e + 1]);
    }
    tmem_st32(taddr_s + c0, sr);
  }
  tmem_st_wait();
  const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
  move_reference<D>(mx, m_ref, l_sum, taddr_o, prev, guard);
  const float nref = m_ref == -INFINITY ? 0.f : -m_ref;
  bool wide = false;
  if (reinterpret_cast<const int*>(scales)[Geometry<D, true>::kCareAt] != 0)   // of all rows alike
    wide = __any_sync(0xffffffffu, mx != -INFINITY && !(l_sum >= need));
  float ps[4] = {0.f, 0.f, 0.f, 0.f};
  if (wide) {
    weights_int8<true>(taddr_s, scales, nref, ps, bars);
  } else {
    weights_int8<false>(taddr_s, scales, nref, ps, bars);
  }
  l_sum += (ps[0] + ps[1]) + (ps[2] + ps[3]);
}

// --------------------------------------------------------------------------------------------
// The kernel
// --------------------------------------------------------------------------------------------

template <typename T, int D, bool kInt8>
__global__ void __launch_bounds__(Geometry<D, kInt8>::kThreads, 1)
    extend_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ CUtensorMap tmq,
                  const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using G = Geometry<D, kInt8>;
  using Sh = Shared<G::kKSlots, G::kVSlots, G::kCodeSlots, G::kScaleSlots, G::kSBufs>;
  constexpr int kSBufs = G::kSBufs;
  constexpr int kKSlots = G::kKSlots, kVSlots = G::kVSlots;
  constexpr int kTileBytes = G::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_smem = smem;
  uint8_t* k_ring = smem + G::kRingOffset;
  uint8_t* v_ring = k_ring + kKSlots * kTileBytes;
  Sh* sh = reinterpret_cast<Sh*>(smem + G::kTailOffset);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  // Warp 0 finds the share, which takes longest: the other preparations are other warps'.
  if (warp == kMmaWarp && lane == 0) {
    sh->abort_flag = 0;
    for (int i = 0; i < kKSlots; ++i) {
      mbar_init(&sh->k_full[i], kInt8 ? 128 : 1);
      mbar_init(&sh->k_empty[i], 1);
    }
    for (int i = 0; i < kVSlots; ++i) {
      mbar_init(&sh->v_full[i], kInt8 ? 128 : 1);
      mbar_init(&sh->v_empty[i], 1);
    }
    for (int i = 0; i < G::kCodeSlots; ++i) {
      mbar_init(&sh->code_full[i], 1);
      mbar_init(&sh->code_empty[i], 128);
    }
    for (int i = 0; i < G::kScaleSlots; ++i) mbar_init(&sh->scale_full[i], 128);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->q_full[t], 1);
      mbar_init(&sh->q_free[t], 1);
      mbar_init(&sh->o_full[t], 1);
    }
    for (int i = 0; i < kSBufs; ++i) {
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_half[i][0], kBM);
      mbar_init(&sh->p_half[i][1], kBM);
    }
    mbar_init(&sh->x_ready, kBM);
    mbar_init(&sh->x_done, kBM);
    mbar_init(&sh->mma_done, 1);
    fence_barrier_init();
  }
  if (warp == kProducerWarp) {
    if (lane == 0) {
      tma_prefetch_desc(&tmq);
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
    __syncwarp();
    tmem_alloc(&sh->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  find_share(a, &sh->share, reinterpret_cast<int*>(k_ring));
  fence_proxy_async_shared();   // the rings were written here; TMA writes it next
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const WaitGuard guard{reinterpret_cast<volatile int*>(&sh->abort_flag), a.status};
  Walk walk;
  Segment s{};

  // Barrier phases run on across segments: each role counts the completions it has waited for.
  if (warp == kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- TMA producer -------------------------------
    // Per segment: Q tile 0, K 0, Q tile 1, K 1, V 0, K 2, V 1, ... Lane i issues copy i of a tile (a
    // part of box_rows cache rows and, at 16 bits, one of the column boxes) from a block it read
    // one tile ahead.
    constexpr int kCols = kInt8 ? 1 : G::kBoxes;
    const int parts = kBN / a.box_rows;
    const bool issues = lane < parts * kCols;
    const int part = lane / kCols, col = lane % kCols;
    const bool paged = a.cache.block_tables != nullptr;
    const uint32_t q_bytes = static_cast<uint32_t>(a.group * a.tile_tokens * D * 2);
    constexpr int kCodeSlots = kInt8 ? G::kCodeSlots : 1;
    int k_issued = 0, v_issued = 0;   // tiles
    int q_loads[2] = {0, 0};
    bool ok = true;
    // Copies the tile at `tile` (this lane's part from block blk) to the next place of its ring.
    auto load = [&](bool is_v, int tile, int blk) -> bool {
      uint64_t *full, *empty;
      uint8_t* dst;
      int n, slots;
      if constexpr (kInt8) {
        n = k_issued + v_issued;
        slots = kCodeSlots;
        full = &sh->code_full[n % slots];
        empty = &sh->code_empty[n % slots];
        dst = smem + G::kCodeOffset + (n % slots) * G::kCodeBytes + part * a.box_rows * D;
      } else {
        n = is_v ? v_issued : k_issued;
        slots = is_v ? kVSlots : kKSlots;
        full = is_v ? &sh->v_full[n % slots] : &sh->k_full[n % slots];
        empty = is_v ? &sh->v_empty[n % slots] : &sh->k_empty[n % slots];
        dst = (is_v ? v_ring : k_ring) + (n % slots) * kTileBytes + col * kBoxBytes +
              part * a.box_rows * 128;
      }
      bool free = n < slots || mbar_wait(empty, ((n / slots) - 1) & 1, guard);
      if (!__all_sync(0xffffffffu, free)) return false;
      if (lane == 0) mbar_arrive_expect_tx(full, kInt8 ? G::kCodeBytes : kTileBytes);
      __syncwarp();
      if (issues) {
        const TmaCoords& c = is_v ? a.vc : a.kc;
        const int key = tile * kBN + part * a.box_rows;
        const int row = paged ? key - a.cache.page.div(key) * a.cache.page.d : key;
        const int once = is_v ? a.v_once : a.k_once;
        const int h = coordinate(s.hkv, once & kOnceHeads), at = coordinate(blk, once & kOnceOuter);
        tma_load_4d(dst, is_v ? &tmv : &tmk, full, col * 64, tma_c(c, 1, row, h, at),
                    tma_c(c, 2, row, h, at), tma_c(c, 3, row, h, at));
      }
      ++(is_v ? v_issued : k_issued);
      return true;
    };
    walk.start(a, sh->share);
    while (ok && walk.next(a, s)) {
      if (s.tiles == 0) continue;
      const int32_t* table = a.cache.block_tables + s.b * a.cache.bt_stride;
      auto block_of = [&](int tile) -> int {
        if (!paged) return s.b;
        const int page = a.cache.page.div(tile * kBN + part * a.box_rows);
        const int blk = issues && page < a.cache.max_blocks ? __ldg(table + page) : -1;
        return blk >= 0 && blk < a.cache.num_blocks ? blk : -1;   // -1 reads as zeros
      };
      auto load_q = [&](int t) -> bool {
        if (s.dual ? t == 1 : s.count(t) == 0) return true;
        if (q_loads[t] > 0 && !mbar_wait(&sh->q_free[t], (q_loads[t] - 1) & 1, guard)) return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->q_full[t], q_bytes);
          for (int box = 0; box < G::kBoxes; ++box)
            tma_load_4d(q_smem + t * kTileBytes + box * kBoxBytes, &tmq, &sh->q_full[t], box * 64, 0,
                        s.hkv, s.seq.row0 + s.first + t * a.tile_tokens);
        }
        ++q_loads[t];
        return true;
      };
      int blk = block_of(s.t0), blk1 = s.t0 + 1 < s.t1 ? block_of(s.t0 + 1) : 0;
      ok = __all_sync(0xffffffffu, load_q(0)) && load(false, s.t0, blk) &&
           __all_sync(0xffffffffu, load_q(1));
      for (int tile = s.t0; ok && tile < s.t1; ++tile) {
        const int blk2 = tile + 2 < s.t1 ? block_of(tile + 2) : 0;
        if (tile + 1 < s.t1) ok = load(false, tile + 1, blk1);
        if (ok) ok = load(true, tile, blk);
        blk = blk1;
        blk1 = blk2;
      }
    }
    // Wait for the copies still landing before the CTA may exit.
    if (lane == 0) {
      auto drain = [&](uint64_t* full, int slots, int issued) {
        for (int i = issued > slots ? issued - slots : 0; i < issued; ++i) {
          if (!mbar_wait(full + i % slots, (i / slots) & 1, guard)) break;
        }
      };
      drain(&sh->q_full[0], 1, q_loads[0]);
      drain(&sh->q_full[1], 1, q_loads[1]);
      if constexpr (kInt8) {
        drain(sh->code_full, kCodeSlots, k_issued + v_issued);
      } else {
        drain(sh->k_full, kKSlots, k_issued);
        drain(sh->v_full, kVSlots, v_issued);
      }
    }
  } else if (warp == kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- MMA issuer -------------------------------
    // One lane waits and issues; the others follow the segments, to help where V rows are zeroed. This
    // lane's own time bounds the kernel once S has a buffer to spare, so a step's places come from few
    // operations and P V and the Q K^T behind it are issued in one go. (All lanes waiting together,
    // with votes, and each step's chain and places from the general formulas: 1450 clocks per step at
    // head_dim 64, whose MMAs take 512.)
    // A one-tile item's second chain reads Q tile 0 as well.
    constexpr int kFmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr int kFmtPv = kInt8 ? 0 : kFmt;
    constexpr uint32_t kIdescQk = umma_idesc_f16(kFmt, kBM, kBN, 0);
    constexpr uint32_t kIdescPv = umma_idesc_f16(kFmtPv, kBM, D, 1);
    const bool leader = elect_one();
    const Desc q_desc(umma_smem_desc_sw128(smem_u32(q_smem), 16, 1024));
    const Desc ring_k(umma_smem_desc_sw128(smem_u32(k_ring), 16, 1024));
    const Desc ring_v(umma_smem_desc_sw128(smem_u32(v_ring), kBoxBytes, 1024));
    int base = 0;                   // key tiles of earlier segments
    int buf = 0, p_parity = 0;      // S buffer of the next step, and the phase of its P
    int q_waits0 = 0, q_waits1 = 0;
    bool ok = true, issued_any = false;
    walk.start(a, sh->share);
    while (ok && walk.next(a, s)) {
      if (s.tiles == 0) continue;
      issued_any = true;
      const int steps = s.count0 + s.count1;
      const int paired = s.paired();
      const int firsts = s.count0 > 0 ? 2 : 1;              // the chains' first steps are i < firsts
      const int last0 = s.other_last();                     // a chain's last step, as is the last one
      auto chain = [&](int i) { return s.chain(i); };
      auto entry_of = [&](int i) {                          // Segment::place, from the first tile on
        return base + (i < paired ? (s.dual ? i : i >> 1) : i - s.count0);
      };
      // Q K^T of step i once its K tile is there; frees what it is the last reader of.
      auto issue_qk = [&](int i, int to) {
        const int c = chain(i), q_tile = s.dual ? 0 : c, slot = entry_of(i) % kKSlots;
        const Desc qd = q_desc.at(q_tile * kTileBytes);
        const Desc kd = ring_k.at(slot * kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(tmem + to * 128, qd.at(kmajor_step(kk)).u64(), kd.at(kmajor_step(kk)).u64(),
                  kIdescQk, kk > 0);
        umma_commit(&sh->s_full[to]);
        if (s.dual || c == 1) umma_commit(&sh->k_empty[slot]);
        if (i == steps - 1 || (!s.dual && i == last0)) umma_commit(&sh->q_free[q_tile]);
      };
      auto wait_k = [&](int i) {
        const int entry = entry_of(i);
        return mbar_wait(&sh->k_full[entry % kKSlots], (entry / kKSlots) & 1, guard);
      };
      auto wait_v = [&](int entry) {
        return mbar_wait(&sh->v_full[entry % kVSlots], (entry / kVSlots) & 1, guard);
      };
      if (leader) {
        for (int i = 0; ok && i < kSBufs && i < steps; ++i) {
          const int c = chain(i);
          if (i < firsts && !(s.dual && c == 1)) {
            ok = mbar_wait(&sh->q_full[c], (c == 0 ? q_waits0 : q_waits1) & 1, guard);
            ++(c == 0 ? q_waits0 : q_waits1);
          }
          ok = ok && wait_k(i);
          tc_fence_after();
          if (ok) issue_qk(i, (buf + i) % kSBufs);
        }
      }
      __syncwarp();
      int zeroed = -1;              // last V entry whose rows past the length were zeroed
      for (int i = 0; i < steps; ++i) {
        const int c = chain(i), entry = entry_of(i), slot = entry % kVSlots;
        if constexpr (!kInt8) {
          const int keys = s.seq.len - (s.t0 + entry - base) * kBN;   // of this tile
          if (keys < kBN && zeroed != entry) {
            zeroed = entry;
            if (leader) ok = ok && wait_v(entry);
            __syncwarp();
            uint8_t* v = v_ring + slot * kTileBytes;
            for (int x = lane; x < (kBN - keys) * 8 * G::kBoxes; x += 32) {
              const int row = keys + x / (8 * G::kBoxes), chunk = x % (8 * G::kBoxes);
              *reinterpret_cast<uint4*>(v + (chunk >> 3) * kBoxBytes + row * 128 +
                                        (chunk & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_shared();
            __syncwarp();
          }
        }
        if (leader && ok) {
          const Desc vd = ring_v.at(slot * kTileBytes);
          const uint32_t accumulate = i >= firsts;
          auto issue_pv = [&](int half) {
#pragma unroll
            for (int kq = 0; kq < kBN / 32; ++kq) {
              const int kk = half * (kBN / 32) + kq;
              umma_ts(tmem + G::kOCol + c * D, tmem + buf * 128 + kk * 8,
                      vd.at(mnmajor_step(kk)).u64(), kIdescPv, kk > 0 ? 1u : accumulate);
            }
          };
          // What the step needs is asked for at once and waited for only where it is missing: four waits
          // in a row cost 100 clocks each when everything is there, which is the usual case.
          const int next = i + kSBufs;   // the step that takes this one's S buffer
          const int next_entry = entry_of(next);
          const bool k_ready = mbar_test_wait(&sh->k_full[next_entry % kKSlots],
                                              (next_entry / kKSlots) & 1);
          const bool v_ready = mbar_test_wait(&sh->v_full[slot], (entry / kVSlots) & 1);
          const bool p0_ready = mbar_test_wait(&sh->p_half[buf][0], p_parity);
          const bool p1_ready = mbar_test_wait(&sh->p_half[buf][1], p_parity);
          ok = (v_ready || wait_v(entry)) &&
               (p0_ready || mbar_wait(&sh->p_half[buf][0], p_parity, guard));
          if (ok) {
            tc_fence_after();
            issue_pv(0);
            if (!p1_ready) {
              ok = mbar_wait(&sh->p_half[buf][1], p_parity, guard);
              tc_fence_after();
            }
          }
          if (ok) {
            issue_pv(1);
            // A two-tile item's V is read last by chain 1, whose tiles are the segment's.
            if (s.dual || c == 1) umma_commit(&sh->v_empty[slot]);
            if (i == last0 || i == steps - 1) umma_commit(&sh->o_full[c]);
            if (next < steps) {
              ok = k_ready || wait_k(next);
              if (ok) issue_qk(next, buf);
            }
          }
        }
        if (++buf == kSBufs) {
          buf = 0;
          p_parity ^= 1;
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      base += s.t1 - s.t0;
    }
    // Every MMA issued has completed before TMEM may be released.
    if (issued_any) {
      if (leader) umma_commit(&sh->mma_done);
      mbar_wait(&sh->mma_done, 0, guard);
    }
  } else if (warp < kProducerWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kSoftmaxRegs));
    // ------------------------------- softmax warpgroups -------------------------------
    const int c = warp >> 2;                  // chain
    const int quarter = warp & 3;             // TMEM lane quarter this warp may access
    const int row = quarter * 32 + lane;      // of the tile
    const uint32_t lane_field = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t taddr_o = tmem + G::kOCol + c * D + lane_field;
    const int row_token = row / a.group;
    const int row_head = row - row_token * a.group;
    int n_base = 0;                           // steps of earlier segments
    int o_waits = 0, joins = 0;
    int kv_base = 0;                          // key tiles of earlier segments
    int segments = 0;
    int4 meta0 = make_int4(0, 0, 0, 0), meta1 = make_int4(0, 0, 0, 0);
    bool ok = true;
    walk.start(a, sh->share);
    while (ok && walk.next(a, s)) {
      const int first_segment = segments++ == 0;
      // This row's token, and whether it holds one.
      const int tile_first = s.dual ? 0 : c * a.tile_tokens;
      const int token = tile_first + row_token;          // within the item
      const bool row_ok = row_token < a.tile_tokens && token < s.tokens;
      const int tile_rows = min(a.tile_tokens, s.tokens - tile_first) * a.group;
      const bool warp_ok = quarter * 32 < tile_rows;     // some row of this warp holds a token
      const int offset = s.seq.len - s.seq.n + s.first;  // position of the item's first token
      const int limit = a.causal ? min(s.seq.len, offset + token + 1) : s.seq.len;
      const int count = s.count(c);

      float m_ref = -INFINITY;  // log2-domain reference point of this row
      float l_sum = 0.f;
      for (int j = 0; j < count; ++j) {
        const int n = n_base + s.order(c, j), buf = n % kSBufs;
        if (!mbar_wait(&sh->s_full[buf], (n / kSBufs) & 1, guard)) {
          ok = false;
          break;
        }
        if (!warp_ok) {   // whatever P holds stays in rows that nobody reads
          tc_fence_after();
          tc_fence_before();
          mbar_arrive(&sh->p_half[buf][0]);
          mbar_arrive(&sh->p_half[buf][1]);
          continue;
        }
        const uint32_t taddr_s = tmem + buf * 128 + lane_field;
        const int v_prev = kv_base + (j > 0 ? s.place(c, j - 1) : 0);
        const PrevPv prev{&sh->v_empty[v_prev % kVSlots],
                          static_cast<uint32_t>((v_prev / kVSlots) & 1),
                          j > 0 && s.order(c, j) - s.order(c, j - 1) < kSBufs};
        tc_fence_after();
        const int k0 = s.tile(c, j) * kBN;
        const bool masked = k0 + kBN > s.seq.len ||
                            (a.causal && k0 + kBN - 1 > offset + tile_first);
        if constexpr (kInt8) {
          const int at = kv_base + s.place(c, j);
          if (!mbar_wait(&sh->scale_full[at % G::kScaleSlots], (at / G::kScaleSlots) & 1, guard)) {
            ok = false;
            break;
          }
          const float* scales = reinterpret_cast<const float*>(smem + G::kScaleOffset) +
                                (at % G::kScaleSlots) * G::kScaleWords;
          softmax_tile_int8<D>(taddr_s, taddr_o, scales, 2.f * count, masked, limit - k0, m_ref,
                               l_sum, sh->p_half[buf], prev, guard);
        } else {
          softmax_tile<T, D>(taddr_s, taddr_o, a.scale_log2, masked, limit - k0, m_ref, l_sum,
                             sh->p_half[buf], prev, guard);
        }
      }
      if (!ok) break;
      kv_base += s.t1 - s.t0;
      n_base += s.count0 + s.count1;

      // The end of the segment. Its O is read before this warpgroup publishes the next segment's
      // first P, which the first P V that overwrites O waits for.
      if (count > 0) {
        if (!mbar_wait(&sh->o_full[c], o_waits & 1, guard)) break;
        ++o_waits;
      }
      float m_other = -INFINITY, l_other = 0.f;
      if (s.joined()) {
        // Chain 1 hands its (m, l) to chain 0, which reads both O and writes the joint result. In an
        // item whose first tile sees no key here the chains only meet: chain 0, which has had no
        // step to wait for, must not reach the next items' barriers ahead of these steps.
        const uint32_t phase = joins++ & 1;
        if (c == 1) {
          sh->x_ml[row] = make_float2(m_ref, l_sum);
          tc_fence_before();
          mbar_arrive(&sh->x_ready);
          if (!mbar_wait(&sh->x_done, phase, guard)) break;
          tc_fence_after();
          if (s.dual) continue;
        } else {
          if (!mbar_wait(&sh->x_ready, phase, guard)) break;
          if (s.dual) {
            const float2 ml = sh->x_ml[row];
            m_other = ml.x;
            l_other = ml.y;
          } else {
            mbar_arrive(&sh->x_done);
          }
        }
      }
      tc_fence_after();
      const bool join = s.count1 > 0 && s.dual;
      const float m = fmaxf(m_ref, m_other);
      const float ref = m == -INFINITY ? 0.f : m;
      float f0 = ex2(m_ref - ref), f1 = ex2(m_other - ref);
      if (!s.dual) f0 = 1.f;
      const float l = s.dual ? scale_sum(l_sum, m_ref - ref) + scale_sum(l_other, m_other - ref) : l_sum;
      const bool whole = s.t0 == 0 && s.t1 == s.tiles;
      if (whole) {
        // A row that saw nothing has l = 0; a NaN sum stays NaN.
        const float inv = l == 0.f ? 0.f : 1.f / l;
        f0 *= inv;
        f1 *= inv;
      }
      const int64_t out_row = s.seq.row0 + s.first + token;
      const int head = s.hkv * a.group + row_head;
      const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
      const int part_row = s.dual ? row : c * kBM + row;
      T* orow = static_cast<T*>(a.o) + out_row * a.o_stride[0] + head * a.o_stride[1];
      float* prow = a.part_o + (static_cast<int64_t>(slot) * (D / 8) * a.part_rows + part_row) * 8;
      if (warp_ok) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t ov[32];
          if (count > 0) {
            tmem_ld32(taddr_o + i * 32, ov);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = 0u;
          }
          float* of = reinterpret_cast<float*>(ov);
#pragma unroll
          for (int e = 0; e < 32; ++e) of[e] *= f0;
          if (join) {
            uint32_t ow[32];
            tmem_ld32(taddr_o + D + i * 32, ow);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) of[e] = fmaf(__uint_as_float(ow[e]), f1, of[e]);
          }
          if (row_ok) {
            if (whole) {
              uint4* dst = reinterpret_cast<uint4*>(orow + i * 32);
#pragma unroll
              for (int v = 0; v < 4; ++v) dst[v] = pack8<T>(of + 8 * v, 1.f);
            } else {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                float4* dst = reinterpret_cast<float4*>(
                    prow + static_cast<int64_t>(i * 4 + v) * a.part_rows * 8);
                dst[0] = make_float4(of[8 * v], of[8 * v + 1], of[8 * v + 2], of[8 * v + 3]);
                dst[1] = make_float4(of[8 * v + 4], of[8 * v + 5], of[8 * v + 6], of[8 * v + 7]);
              }
            }
          }
        }
      }
      tc_fence_before();
      if (s.dual) mbar_arrive(&sh->x_done);
      if (row_ok) {
        if (whole) {
          a.lse[out_row * a.heads + head] =
              l == 0.f ? -INFINITY : m * 0.69314718055994530942f + logf(l);
        } else {
          reinterpret_cast<float2*>(a.part_ml)[static_cast<int64_t>(slot) * a.part_rows + part_row] =
              make_float2(m, l);
        }
      }
      if (!whole) {
        const int4 meta = make_int4(kPartValid | (s.t0 == 0 ? kPartOpens : 0) |
                                        (s.t1 == s.tiles ? kPartCloses : 0),
                                    s.seq.row0 + s.first, s.tokens, s.hkv);
        if (first_segment) meta0 = meta;
        else meta1 = meta;
      }
    }
    if (threadIdx.x == 0) {
      a.part_meta[2 * blockIdx.x] = meta0;
      a.part_meta[2 * blockIdx.x + 1] = meta1;
    }
  } else if (warp >= kConvertWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    if constexpr (kInt8) {
      // ------------------------------- code converters -------------------------------
      // One warpgroup for K, one for V. Code tiles are copied in the producer's order (code_place).
      const bool is_v = warp >= kConvertWarp + 4;
      const int tid = threadIdx.x - (is_v ? kConvertWarp + 4 : kConvertWarp) * 32;
      const bool paged = a.cache.block_tables != nullptr;
      int base = 0;   // key tiles of earlier segments
      bool ok = true;
      // Key tile i of the segment, once it and its place in the 16-bit ring are there.
      auto convert = [&](int i, int n) -> bool {
        const int code = 2 * base + code_place(is_v, i, n);
        const int code_slot = code % G::kCodeSlots, code_phase = code / G::kCodeSlots;
        // The place's last tile may have been the other warpgroup's: its release says that the phase
        // of code_full before this one has completed.
        if (code_phase > 0 && !mbar_wait(&sh->code_empty[code_slot], (code_phase - 1) & 1, guard))
          return false;
        if (!mbar_wait(&sh->code_full[code_slot], code_phase & 1, guard)) return false;
        const int at = base + i, slots = is_v ? kVSlots : kKSlots, slot = at % slots;
        uint64_t* empty = is_v ? &sh->v_empty[slot] : &sh->k_empty[slot];
        if (at >= slots && !mbar_wait(empty, ((at / slots) - 1) & 1, guard)) return false;
        const uint8_t* codes = smem + G::kCodeOffset + code_slot * G::kCodeBytes;
        if (is_v) {
          convert_tile<__half, D>(codes, v_ring + slot * kTileBytes, tid);
        } else {
          convert_tile<T, D>(codes, k_ring + slot * kTileBytes, tid);
        }
        fence_proxy_async_shared();
        mbar_arrive(is_v ? &sh->v_full[slot] : &sh->k_full[slot]);
        mbar_arrive(&sh->code_empty[code_slot]);
        return true;
      };
      walk.start(a, sh->share);
      while (ok && walk.next(a, s)) {
        const int n = s.t1 - s.t0;
        if (is_v) {
          for (int i = 0; ok && i < n; ++i) ok = convert(i, n);
          base += n;
          continue;
        }
        // Thread r of the K warpgroup also holds key r of the tile: its scales are read one tile
        // ahead, its block two.
        const int32_t* table = a.cache.block_tables + s.b * a.cache.bt_stride;
        auto block_of = [&](int tile) -> int {
          if (!paged) return s.b;
          const int page = a.cache.page.div(tile * kBN + tid);
          const int blk = page < a.cache.max_blocks ? __ldg(table + page) : -1;
          return blk < a.cache.num_blocks ? blk : -1;
        };
        auto scales_of = [&](int tile, int blk, float& sk, float& sv) {
          const int key = tile * kBN + tid;
          sk = 0.f;
          sv = kMinScale;
          if (key < s.seq.len && blk >= 0) {
            const int64_t r = paged ? key - a.cache.page.div(key) * a.cache.page.d : key;
            sk = a.cache.ks[blk * a.cache.ks_stride[0] + r * a.cache.ks_stride[1] +
                            s.hkv * a.cache.ks_stride[2]];
            sv = a.cache.vs[blk * a.cache.vs_stride[0] + r * a.cache.vs_stride[1] +
                            s.hkv * a.cache.vs_stride[2]];
          }
        };
        float sk = 0.f, sv = 0.f;
        int blk_next = 0;
        bool care = false;   // these keys of the segment had a V scale out of the ordinary
        if (n > 0) {
          scales_of(s.t0, block_of(s.t0), sk, sv);
          blk_next = block_of(s.t0 + 1);
        }
        for (int i = 0; ok && i < n; ++i) {
          float sk_next = 0.f, sv_next = 0.f;
          if (i + 1 < n) {
            scales_of(s.t0 + i + 1, blk_next, sk_next, sv_next);
            blk_next = block_of(s.t0 + i + 2);
          }
          // The place of these scales is free once K 's is (see kScaleSlots).
          const int at = base + i;
          if (at >= kKSlots &&
              !mbar_wait(&sh->k_empty[at % kKSlots], ((at / kKSlots) - 1) & 1, guard)) {
            ok = false;
            break;
          }
          float* out = reinterpret_cast<float*>(smem + G::kScaleOffset) +
                       (at % G::kScaleSlots) * G::kScaleWords;
          // Keys past the length have no weight.
          const bool in = (s.t0 + i) * kBN + tid < s.seq.len;
          const bool finite = sv <= kMaxScale;
          // A V scale that is not finite makes the score NaN: it reaches the rows that see the key
          // and adds nothing to the sums of the others.
          out[tid] = !in ? 0.f : finite ? sk * a.scale_log2 : __int_as_float(0x7fffffff);
          sv = fmaxf(sv, kMinScale);
          const float log2_sv = !in ? -INFINITY : finite ? __log2f(sv) : 0.f;
          out[kBN + tid] = log2_sv;
          out[2 * kBN + tid] = in && finite ? 1.f / sv : 0.f;
          care = care || __any_sync(0xffffffffu, in && !(log2_sv >= -40.f && log2_sv <= 45.f));
          if ((tid & 31) == 0) reinterpret_cast<uint8_t*>(out + G::kCareAt)[tid >> 5] = care ? 1 : 0;
          mbar_arrive(&sh->scale_full[at % G::kScaleSlots]);
          sk = sk_next;
          sv = sv_next;
          ok = convert(i, n);
        }
        base += n;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- warps 10 and 11 -------------------------------
    zero_other_rows<T, D>(a, blockIdx.x * 2 + warp - 10, gridDim.x * 2, lane);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of the items that were cut, of one launch or (blocks past the first `ctas`) of
// two. Block (c, y) handles the item that CTA c opened without closing, if there is one: its parts
// are that slot and the first slots of the following CTAs, up to the one that closes it, combined
// in that order (CTAs whose share held no whole key tile of the item left none). A thread owns 8
// columns of one row.
// kBatch parts' loads are issued together: 8 for launches of few rows, whose items are cut into many
// parts, 4 (four blocks per SM) for large partials, where most blocks only find nothing to do. It is
// bound by its chain of dependent L2 loads (flags, then parts): 5 us after a few-row launch, 7-11 us
// after one of two-tile items.
template <typename T, int D, int kBatch>
__global__ void __launch_bounds__(256, kBatch == 4 ? 4 : 2) extend_merge_kernel(
    const __grid_constant__ ExtendArgs first, const __grid_constant__ ExtendArgs second, int ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bool is_first = static_cast<int>(blockIdx.x) < ctas;
  const ExtendArgs& a = is_first ? first : second;
  __shared__ int first_flags[kMaxCtas];   // flags of the CTAs' first slots
  const int cta = is_first ? blockIdx.x : blockIdx.x - ctas;
  int open = -1;
  int4 meta = make_int4(0, 0, 0, 0);
  if (static_cast<int>(blockIdx.y) * 256 >= a.part_rows * (D / 8)) return;
  const int4 m0 = a.part_meta[2 * cta], m1 = a.part_meta[2 * cta + 1];
  constexpr int kWhich = kPartValid | kPartOpens | kPartCloses;
  if ((m0.x & kWhich) == (kPartValid | kPartOpens)) {
    open = 2 * cta;
    meta = m0;
  } else if ((m1.x & kWhich) == (kPartValid | kPartOpens)) {
    open = 2 * cta + 1;
    meta = m1;
  }
  if (open < 0) return;
  for (int i = cta + 1 + threadIdx.x; i < ctas; i += 256) first_flags[i] = a.part_meta[2 * i].x;
  __syncthreads();
  const int idx = blockIdx.y * 256 + threadIdx.x;
  const int row = idx % a.part_rows, col = idx / a.part_rows;
  const int in_tile = row % kBM, tile = row / kBM;
  const int tile_token = in_tile / a.group;
  const int token = tile * a.tile_tokens + tile_token;
  if (col >= D / 8 || tile_token >= a.tile_tokens || token >= meta.z) return;

  float m = -INFINITY, l = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  int slot = open, next = cta + 1;
  auto following = [&]() -> int {   // the next part's slot, -1 past the one that closes the item
    while (next < ctas) {
      const int flags = first_flags[next], at = 2 * next;
      ++next;
      if (flags & kPartValid) {
        if (flags & kPartCloses) next = ctas;
        return at;
      }
    }
    return -1;
  };
  while (slot >= 0) {
    float2 ml[kBatch];
    float4 o0[kBatch], o1[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      o0[i] = o1[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (slot >= 0) {
        ml[i] = reinterpret_cast<const float2*>(a.part_ml)[static_cast<int64_t>(slot) * a.part_rows +
                                                           row];
        const float4* src = reinterpret_cast<const float4*>(
            a.part_o + ((static_cast<int64_t>(slot) * (D / 8) + col) * a.part_rows + row) * 8);
        o0[i] = src[0];
        o1[i] = src[1];
        slot = following();
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (ml[i].x != -INFINITY) {
        const float m_new = fmaxf(m, ml[i].x);
        const float keep = ex2(m - m_new), f = ex2(ml[i].x - m_new);
        l = scale_sum(l, m - m_new) + scale_sum(ml[i].y, ml[i].x - m_new);
        m = m_new;
        acc[0] = acc[0] * keep + o0[i].x * f;
        acc[1] = acc[1] * keep + o0[i].y * f;
        acc[2] = acc[2] * keep + o0[i].z * f;
        acc[3] = acc[3] * keep + o0[i].w * f;
        acc[4] = acc[4] * keep + o1[i].x * f;
        acc[5] = acc[5] * keep + o1[i].y * f;
        acc[6] = acc[6] * keep + o1[i].z * f;
        acc[7] = acc[7] * keep + o1[i].w * f;
      } else {
        l += ml[i].y;   // no weight: 0, or NaN when every score of the part was NaN
      }
    }
  }
  const int64_t out_row = meta.y + token;
  const int head = meta.w * a.group + (in_tile - tile_token * a.group);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* dst = static_cast<T*>(a.o) + out_row * a.o_stride[0] + head * a.o_stride[1] + col * 8;
  *reinterpret_cast<uint4*>(dst) = pack8<T>(acc, inv);
  if (col == 0)
    a.lse[out_row * a.heads + head] = l == 0.f ? -INFINITY
                                               : m * 0.69314718055994530942f + logf(l);
}

// --------------------------------------------------------------------------------------------
// Host
// --------------------------------------------------------------------------------------------

template <typename T, int D, bool kInt8>
int launch(const ExtendArgs& a, const CUtensorMap& tmq, const CUtensorMap& tmk,
           const CUtensorMap& tmv, int ctas, int dev, cudaStream_t stream) {
  using G = Geometry<D, kInt8>;
  constexpr int kSmem = G::kTailOffset + static_cast<int>(sizeof(Shared<G::kKSlots, G::kVSlots, G::kCodeSlots,
                                                               G::kScaleSlots, G::kSBufs>)) +
                        1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
  auto kernel = extend_kernel<T, D, kInt8>;
  static thread_local int configured_device = -1;
  if (configured_device != dev) {
    if (int st = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSmem),
                            "cudaFuncSetAttribute(extend)"))
      return st;
    // setmaxnreg.inc would wait forever in a build launched with fewer registers than the split.
    cudaFuncAttributes attr{};
    if (int st = check_cuda(cudaFuncGetAttributes(&attr, kernel), "cudaFuncGetAttributes(extend)"))
      return st;
    if (attr.numRegs * G::kThreads < 256 * G::kSoftmaxRegs + (G::kThreads - 256) * G::kOtherRegs)
      return fail(FLB_ERR_CUDA, "extend kernel built with %d registers per thread, fewer than its "
                  "register split needs", attr.numRegs);
    configured_device = dev;
  }
  kernel<<<ctas, G::kThreads, kSmem, stream>>>(a, tmq, tmk, tmv);
  return check_cuda(cudaGetLastError(), "extend_kernel launch");
}

constexpr int kFewPartRows = 64;   // rows of a partial up to which a merge has few blocks

// Merges the partials of `count` (1 or 2) launches.
template <typename T, int D>
int launch_merge(const ExtendArgs* a, int count, int ctas, cudaStream_t stream) {
  const int rows = std::max(a[0].part_rows, a[count - 1].part_rows);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(count * ctas, (rows * (D / 8) + 255) / 256);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];   // scheduled while the last launch drains
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kernel = rows <= kFewPartRows ? extend_merge_kernel<T, D, 8> : extend_merge_kernel<T, D, 4>;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a[0], a[count - 1], ctas),
                    "extend_merge_kernel launch");
}

template <typename T>
int launch_merge_t(int head_dim, const ExtendArgs* a, int count, int ctas, cudaStream_t stream) {
  return head_dim == 128 ? launch_merge<T, 128>(a, count, ctas, stream)
                         : launch_merge<T, 64>(a, count, ctas, stream);
}

template <typename T>
int launch_t(const flb_kv_cache* c, const ExtendArgs& a, const CUtensorMap& tmq,
             const CUtensorMap& tmk, const CUtensorMap& tmv, int ctas, int dev, cudaStream_t s) {
  const bool int8 = c->dtype == FLB_INT8;
  if (c->head_dim == 128)
    return int8 ? launch<T, 128, true>(a, tmq, tmk, tmv, ctas, dev, s)
                : launch<T, 128, false>(a, tmq, tmk, tmv, ctas, dev, s);
  return int8 ? launch<T, 64, true>(a, tmq, tmk, tmv, ctas, dev, s)
              : launch<T, 64, false>(a, tmq, tmk, tmv, ctas, dev, s);
}

// Rows of a partial: the most score rows an item can have.
int part_rows(int64_t rows, int group) {
  const int tile_tokens = kBM / group;
  return rows <= tile_tokens ? static_cast<int>(rows) * group : 2 * kBM;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

int validate(const flb_kv_cache* c, const flb_extend_params* p) {
  if (int st = validate_kv_cache(c)) return st;
  if (p == nullptr) return fail(FLB_ERR_INVALID_ARGUMENT, "params is NULL");
  if (!p->q || !p->o || !p->lse || !p->seq_lens)
    return fail(FLB_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (p->rows <= 0 || p->heads <= 0 || (p->cu_seqlens == nullptr && p->rows_per_seq <= 0))
    return fail(FLB_ERR_INVALID_ARGUMENT, "empty input: %d rows, %d per sequence, %d heads",
                p->rows, p->rows_per_seq, p->heads);
  if (p->heads % c->heads_kv != 0)
    return fail(FLB_ERR_INVALID_ARGUMENT,
                "the number of query heads (%d) must be a multiple of KV heads (%d)", p->heads,
                c->heads_kv);
  if (p->heads / c->heads_kv > kBM)
    return fail(FLB_ERR_UNSUPPORTED, "more than %d query heads per KV head", kBM);
  if (p->dtype != FLB_BF16 && p->dtype != FLB_FP16)
    return fail(FLB_ERR_UNSUPPORTED, "extend takes bf16 or fp16 queries (dtype code %d)", p->dtype);
  if (c->dtype != FLB_INT8 && c->dtype != p->dtype)
    return fail(FLB_ERR_UNSUPPORTED, "queries (dtype code %d) and cache (%d) differ", p->dtype,
                c->dtype);
  if (!(p->softmax_scale > 0.f) || !(p->softmax_scale <= 3.0e38f))
    return fail(FLB_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and finite");
  const int cache_rows = c->block_tables != nullptr ? c->page_size : c->max_seqlen;
  if ((p->rows > 1 && (p->q_row_stride == 0 || p->o_row_stride == 0)) ||
      (p->heads > 1 && (p->q_head_stride == 0 || p->o_head_stride == 0)) ||
      (cache_rows > 1 && (c->k_seq_stride == 0 || c->v_seq_stride == 0)))
    return fail(FLB_ERR_UNSUPPORTED,
                "rows and heads of q and o, and keys, must lie apart: found a stride 0");
  const int ps = c->page_size;
  if (c->block_tables != nullptr && !(ps == 8 || ps == 16 || ps == 32 || ps % 64 == 0))
    return fail(FLB_ERR_UNSUPPORTED, "paged cache: page_size %d must be 8, 16, 32 or a multiple of 64",
                ps);
  if (c->batch > kMaxBatch)
    return fail(FLB_ERR_UNSUPPORTED, "more than %d sequences in one call", kMaxBatch);
  // Units of one KV head (extend_work.cuh) must fit in 31 bits.
  const int tile_tokens = kBM / (p->heads / c->heads_kv);
  const int64_t items = p->rows / (2 * tile_tokens) + c->batch;
  const int64_t max_units = items * (kItemUnits + 2 * ((c->max_seqlen + int64_t{kBN} - 1) / kBN));
  if (max_units > 0x7fffffffLL)
    return fail(FLB_ERR_UNSUPPORTED, "problem too large for one launch");
  const View4 qv{p->q, {1, p->rows, p->heads, c->head_dim},
                 {0, p->q_row_stride, p->q_head_stride, 1}, 2};
  const View4 ov{p->o, {1, p->rows, p->heads, c->head_dim},
                 {0, p->o_row_stride, p->o_head_stride, 1}, 2};
  if (!rows_16b_aligned(qv))
    return fail(FLB_ERR_MISALIGNED, "q must have 16-byte aligned rows (data pointer and strides)");
  if (!rows_16b_aligned(ov))
    return fail(FLB_ERR_MISALIGNED, "o must have 16-byte aligned rows (data pointer and strides)");
  return FLB_OK;
}

}  // namespace
}  // namespace flb

using namespace flb;

namespace {

// The partials of one launch: metadata, (m, l), O.
size_t partial_bytes(size_t ctas, size_t rows, size_t head_dim) {
  return align256(2 * ctas * sizeof(int4)) + align256(2 * ctas * rows * 2 * sizeof(float)) +
         align256(2 * ctas * rows * head_dim * sizeof(float));
}

void set_partials(ExtendArgs* a, char* ws, size_t ctas, int rows) {
  a->part_rows = rows;
  a->part_meta = reinterpret_cast<int4*>(ws);
  ws += align256(2 * ctas * sizeof(int4));
  a->part_ml = reinterpret_cast<float*>(ws);
  ws += align256(2 * ctas * static_cast<size_t>(rows) * 2 * sizeof(float));
  a->part_o = reinterpret_cast<float*>(ws);
}

// Cache rows of one TMA box: whole tiles of a contiguous cache, else rows that never cross a page.
int box_rows_for(const flb_kv_cache* c) {
  return c->block_tables == nullptr || c->page_size % kBN == 0 ? kBN : std::min(c->page_size, 64);
}

}  // namespace

extern "C" size_t flb_extend_workspace_bytes(int32_t rows, int32_t heads, int32_t heads_kv,
                                             int32_t head_dim, int32_t sm_count) {
  if (rows <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 ||
      heads / heads_kv > kBM || head_dim <= 0 || sm_count <= 0)
    return 0;
  // Both kernels of a call over an int8 cache have partials of their own.
  return partial_bytes(sm_count, kFewTile, head_dim) +
         partial_bytes(sm_count, part_rows(rows, heads / heads_kv), head_dim);
}

extern "C" int flb_extend_fwd(const flb_kv_cache* c, const flb_extend_params* p,
                              flb_stream_t stream_) {
  clear_error();
  if (int st = validate(c, p)) return st;
  int dev = 0, sm_count = 0;
  if (int st = current_device_info(&dev, &sm_count, nullptr, nullptr)) return st;
  if (sm_count > kMaxCtas) return fail(FLB_ERR_UNSUPPORTED, "more than %d SMs", kMaxCtas);
  const size_t need =
      flb_extend_workspace_bytes(p->rows, p->heads, c->heads_kv, c->head_dim, sm_count);
  if (p->workspace == nullptr || p->workspace_bytes < need)
    return fail(FLB_ERR_WORKSPACE, "extend needs %zu bytes of workspace, got %zu", need,
                p->workspace == nullptr ? size_t{0} : p->workspace_bytes);
  if (reinterpret_cast<uintptr_t>(p->workspace) % 16 != 0)
    return fail(FLB_ERR_MISALIGNED, "the workspace must be 16-byte aligned");

  ExtendArgs a{};
  a.o = p->o;
  a.lse = p->lse;
  a.o_stride[0] = p->o_row_stride;
  a.o_stride[1] = p->o_head_stride;
  a.seq_lens = p->seq_lens;
  a.ragged = Ragged{p->cu_seqlens, p->rows, p->rows_per_seq, c->batch};
  a.status = p->status;
  a.heads = p->heads;
  a.group = p->heads / c->heads_kv;
  a.causal = p->causal ? 1 : 0;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->softmax_scale) * 1.4426950408889634);
  a.cache = kv_view(c);
  a.box_rows = box_rows_for(c);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  char* ws = static_cast<char*>(p->workspace);
  ExtendArgs done[2];   // launches whose partials are to be merged
  int launches = 0;
  auto merge = [&] {
    return p->dtype == FLB_BF16
               ? launch_merge_t<__nv_bfloat16>(c->head_dim, done, launches, sm_count, stream)
               : launch_merge_t<__half>(c->head_dim, done, launches, sm_count, stream);
  };

  // Which kernel: by the rows of every sequence when they are known here, else both (int8).
  const bool int8 = c->dtype == FLB_INT8;
  const bool known = p->cu_seqlens == nullptr || c->batch == 1;
  const int64_t per_seq = p->cu_seqlens == nullptr ? p->rows_per_seq : p->rows;
  const bool few = int8 && a.group <= kFewTile && (!known || per_seq <= kFewTile / a.group);
  const bool many = !few || !known;
  if (few) {
    ExtendArgs f = a;
    // With unknown row counts, up to 8 score rows per sequence where the group allows it: the form
    // of single tokens, which is the faster one by a third.
    f.tile_tokens = !many                  ? static_cast<int>(per_seq)
                    : a.group <= kFewTile / 2 ? kFewTile / 2 / a.group
                                              : 1;
    f.few_tokens = a.few_tokens = f.tile_tokens;
    f.select = many ? kFewRows : kAllRows;
    f.item_tokens = FastDiv::of(2 * f.tile_tokens);
    set_partials(&f, ws, sm_count, kFewTile);
    if (int st = launch_extend_few(f, c, p->q, p->q_row_stride, p->q_head_stride, p->dtype,
                                   sm_count, dev, stream))
      return st;
    done[launches++] = f;
  }
  if (!many) return merge();
  a.tile_tokens = kBM / a.group;
  a.item_tokens = FastDiv::of(2 * a.tile_tokens);
  a.select = few ? kManyRows : kAllRows;
  set_partials(&a, ws + partial_bytes(sm_count, kFewTile, c->head_dim), sm_count,
               part_rows(p->rows, a.group));
  CUtensorMap tmq, tmk, tmv;
  View4 kv = kv_view4(c, false), vv = kv_view4(c, true);
  a.k_once = fold_expanded(&kv);
  a.v_once = fold_expanded(&vv);
  if (int8) {
    if (int st = encode_rows_map(&tmk, &a.kc, kv, a.box_rows, c->head_dim, FLB_INT8, 0)) return st;
    if (int st = encode_rows_map(&tmv, &a.vc, vv, a.box_rows, c->head_dim, FLB_INT8, 0)) return st;
  } else {
    if (int st = encode_rows_x64_map(&tmk, &a.kc, kv, a.box_rows, c->dtype)) return st;
    if (int st = encode_rows_x64_map(&tmv, &a.vc, vv, a.box_rows, c->dtype)) return st;
  }
  if (int st = encode_group_map(&tmq, p->q, p->rows, c->heads_kv, a.group, c->head_dim,
                                p->q_row_stride, p->q_head_stride, a.tile_tokens, p->dtype))
    return st;
  const int st = p->dtype == FLB_BF16
                     ? launch_t<__nv_bfloat16>(c, a, tmq, tmk, tmv, sm_count, dev, stream)
                     : launch_t<__half>(c, a, tmq, tmk, tmv, sm_count, dev, stream);
  if (st != FLB_OK) return st;
  done[launches++] = a;
  return merge();
}
