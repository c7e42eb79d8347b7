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
// scales, and no rounding beyond theirs is made.
//
// What bounds it. Every K/V byte is read once per 2 x 128 rows, so few rows per sequence are bound
// by HBM (2 H_kv D bytes per key at 8 bits, twice that at 16) and chunks of hundreds of rows by the
// tensor cores and the exponentials.
//
// How it is split.
//  * A tile of 128 score rows is (tokens x the query heads of one KV head): head h of token i is
//    row i * group + h, so K/V are read once per group and a few tokens fill a tile. Q comes by
//    TMA as a [64 columns x group x tokens] box.
//  * An item is two such tiles of one (sequence, KV head), one softmax warpgroup each, over the keys
//    its last row sees. When its tokens fit in one tile, both warpgroups work on that tile, on
//    alternate key tiles (a chain of Q K^T, softmax, P V is latency bound: two of them per SM are
//    twice the rate), and the first joins the two results through TMEM at the end.
//  * One CTA per SM. The items' key tiles, in the order (sequence, KV head, item, key tile), are cut
//    into equal shares (a tile of a two-tile item counts twice, and each item has a fixed part), so
//    a long cache with few rows spreads over all SMs and ragged batches stay balanced. Every CTA
//    finds its share from cu_seqlens and seq_lens on the device. An item that is cut leaves fp32
//    partials (at most two per CTA) that extend_merge_kernel joins in key order.
//  * Warps: two softmax warpgroups, a TMA producer, the MMA issuer, and for int8 a warpgroup that
//    turns [128 x D] code tiles into the 16-bit tiles the tensor cores read.
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

#include "kv_cache.cuh"
#include "sm100.cuh"

namespace flb {
namespace {

constexpr int kBM = 128;              // score rows per tile
constexpr int kBN = 128;              // keys per tile
constexpr int kBoxBytes = kBM * 128;  // a swizzled [128 rows x 64 columns] 16-bit box
constexpr uint32_t kTmemCols = 512;   // S0 | S1 | O0 | O1
constexpr float kRescaleThreshold = 8.0f;   // log2 units: weights stay <= 2^8
constexpr int kItemUnits = 2;         // fixed cost of an item, in halves of a two-tile key tile
constexpr int kMaxBatch = 8192;       // the units' prefix sums use the K/V ring before it fills
constexpr float kMinScale = 0x1p-100f;
constexpr int kMaxCtas = 256;         // SMs of a device (one CTA each)
constexpr int kScaleSlots = 4;        // key tiles whose scales are held (see the converter)

constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kConvertWarp = 12;      // int8: warps 12-15

// 16-bit: 128 KB of K/V tiles beside the two Q tiles. int8: 96 KB of 16-bit tiles, 48 KB of codes.
template <int D, bool kInt8>
struct Geometry {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  static constexpr int kBoxes = D / 64;
  static constexpr int kTileBytes = kBM * D * 2;
  static constexpr int kCodeBytes = kBN * D;
  static constexpr int kSlots = (kInt8 ? 3 : 4) * (128 / D);
  static constexpr int kCodeSlots = kInt8 ? 3 * (128 / D) : 0;
  static constexpr int kScaleBytes = kInt8 ? kScaleSlots * 3 * kBN * 4 : 0;
  static constexpr int kRingOffset = 2 * kTileBytes;
  static constexpr int kCodeOffset = kRingOffset + kSlots * kTileBytes;
  static constexpr int kScaleOffset = kCodeOffset + kCodeSlots * kCodeBytes;
  static constexpr int kTailOffset = kScaleOffset + kScaleBytes;
  static constexpr int kThreads = kInt8 ? 512 : 384;
  // The register split (setmaxnreg) must not exceed what the CTA is launched with.
  static constexpr int kLaunchRegs = kInt8 ? 128 : 168;
  static constexpr int kSoftmaxRegs = kInt8 ? 200 : 216;
  static constexpr int kOtherRegs = kInt8 ? 56 : 72;
  static_assert(2 * 128 * kSoftmaxRegs + (kThreads - 256) * kOtherRegs <= kThreads * kLaunchRegs,
                "the register split must fit in the launch's registers");
  static_assert((kMaxBatch + 1) * 8 <= kSlots * kTileBytes, "prefix sums fit in the ring");
};

struct ExtendArgs {
  void* o;
  float* lse;
  int64_t o_stride[2];                // row, head
  const int32_t* seq_lens;
  Ragged ragged;
  int* status;
  int heads, group, causal;
  int tile_tokens;                    // tokens per tile: 128 / group
  int box_rows;                       // cache rows per TMA box (a box never crosses a page)
  float scale_log2;
  TmaCoords kc, vc;
  // Partials: slot 2 c + i is CTA c's first (0) or last (1) item share. part_o holds
  // [slots][D / 8][part_rows][8], part_ml [slots][part_rows][2].
  int part_rows;
  float* part_o;
  float* part_ml;
  int4* part_meta;                    // [slots]: flags, first token's row, tokens, KV head
  KvView cache;
};

enum : int { kPartValid = 1, kPartOpens = 2, kPartCloses = 4 };

template <int kSlots, int kCodeSlots>
struct Shared {
  uint64_t q_full[2];
  uint64_t q_free[2];        // the last Q K^T of an item that reads a Q tile has completed
  uint64_t kv_full[kSlots];
  uint64_t kv_empty[kSlots];
  uint64_t code_full[kCodeSlots + 1];
  uint64_t code_empty[kCodeSlots + 1];
  uint64_t scale_full[kScaleSlots];
  uint64_t s_full[2];
  uint64_t p_half[2][2];     // P of keys 0-63 / 64-127 of a tile stored in TMEM
  uint64_t o_full[2];
  uint64_t x_ready, x_done;  // joining the two chains of a one-tile item
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
  int start[4];              // where this CTA's share starts: sequence, KV head, item, unit in it
  int64_t units;             // and how long it is
  float2 x_ml[kBM];          // (m, l) of the second chain's rows
};

__device__ __forceinline__ int tma_c(const TmaCoords& c, int slot, int s, int h, int b) {
  return c.pos_s == slot ? s : (c.pos_h == slot ? h : b);
}

// --------------------------------------------------------------------------------------------
// The work
// --------------------------------------------------------------------------------------------

struct Sequence {
  int row0, n, len;   // first row, rows, keys
};

__device__ __forceinline__ Sequence load_sequence(const ExtendArgs& a, int b) {
  Sequence s;
  const Ragged& r = a.ragged;
  int end;
  if (r.cu != nullptr) {
    s.row0 = min(max(__ldg(r.cu + b), 0), r.rows);
    end = min(max(__ldg(r.cu + b + 1), s.row0), r.rows);
  } else {
    s.row0 = static_cast<int>(min(static_cast<int64_t>(b) * r.rows_per_seq,
                                  static_cast<int64_t>(r.rows)));
    end = s.row0 + min(r.rows_per_seq, r.rows - s.row0);
  }
  s.n = end - s.row0;
  s.len = min(max(__ldg(a.seq_lens + b), 0), a.cache.max_seqlen);
  return s;
}

// Key tiles that the first `tokens` rows of a sequence see.
__device__ __forceinline__ int tiles_seen(const ExtendArgs& a, const Sequence& s, int tokens) {
  const int keys = a.causal ? min(s.len, s.len - s.n + tokens) : s.len;
  return keys <= 0 ? 0 : (keys + kBN - 1) / kBN;
}

// Item k of a sequence: tokens [k 2 tt, (k + 1) 2 tt). Its cost in units.
__device__ __forceinline__ int items_of(const ExtendArgs& a, const Sequence& s) {
  return (s.n + 2 * a.tile_tokens - 1) / (2 * a.tile_tokens);
}
__device__ __forceinline__ int item_units(const ExtendArgs& a, const Sequence& s, int k) {
  const int first = k * 2 * a.tile_tokens;
  const int last = min(first + 2 * a.tile_tokens, s.n);
  const int weight = last - first <= a.tile_tokens ? 1 : 2;
  return kItemUnits + weight * tiles_seen(a, s, last);
}

// A CTA's part of an item: key tiles [t0, t1) of all `tiles`.
struct Segment {
  Sequence seq;
  int b, hkv, first, tokens;   // sequence, KV head, first token in it, tokens
  int t0, t1, tiles;
  bool dual;                   // the tokens fit in one tile
  int count[2];                // key tiles each chain runs here

  // Chain c's j-th key tile.
  __device__ __forceinline__ int tile(int c, int j) const { return dual ? t0 + 2 * j + c : t0 + j; }
  // Its place in this segment's ring order.
  __device__ __forceinline__ int place(int c, int j) const { return dual ? 2 * j + c : j; }
};

// Walks a CTA's share segment by segment; every role walks the same sequence of segments.
struct Walk {
  Sequence seq;
  int b, hkv, k, at;
  int64_t left;

  template <typename Sh>
  __device__ __forceinline__ void start(const ExtendArgs& a, const Sh* sh) {
    b = sh->start[0];
    hkv = sh->start[1];
    k = sh->start[2];
    at = sh->start[3];
    left = sh->units;
    if (left > 0) seq = load_sequence(a, b);
  }

  __device__ __forceinline__ bool next(const ExtendArgs& a, Segment& s) {
    while (left > 0) {
      const int per_item = 2 * a.tile_tokens;
      s.seq = seq;
      s.b = b;
      s.hkv = hkv;
      s.first = k * per_item;
      s.tokens = min(per_item, seq.n - s.first);
      s.dual = s.tokens <= a.tile_tokens;
      s.tiles = tiles_seen(a, seq, s.first + s.tokens);
      const int weight = s.dual ? 1 : 2;
      const int total = kItemUnits + weight * s.tiles;
      const int from = at;
      const int to = static_cast<int>(min(static_cast<int64_t>(total), at + left));
      s.t0 = (max(from - kItemUnits, 0) + weight - 1) / weight;
      s.t1 = (max(to - kItemUnits, 0) + weight - 1) / weight;
      left -= to - from;
      at = to;
      if (to == total) {
        at = 0;
        if (++k >= items_of(a, seq)) {
          k = 0;
          if (++hkv >= a.cache.heads_kv) {
            hkv = 0;
            if (left > 0) {
              do {
                seq = load_sequence(a, ++b);
              } while (seq.n == 0);   // some later sequence has rows: units are left
            }
          }
        }
      }
      if (s.t1 > s.t0 || (s.tiles == 0 && from == 0)) {
        const int n = s.t1 - s.t0;
        if (s.dual) {
          s.count[0] = (n + 1) / 2;
          s.count[1] = n / 2;
        } else {
          s.count[0] = min(max(tiles_seen(a, s.seq, s.first + a.tile_tokens), s.t0), s.t1) - s.t0;
          s.count[1] = n;
        }
        return true;
      }
    }
    return false;
  }
};

// Finds this CTA's share. All threads; `pref` is shared memory for batch + 1 values.
template <typename Sh>
__device__ __forceinline__ void find_share(const ExtendArgs& a, Sh* sh, int64_t* pref) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int batch = a.ragged.batch;
  constexpr int kFew = 4;   // items one thread sums by itself
  for (int b = threadIdx.x; b < batch; b += blockDim.x) {
    const Sequence s = load_sequence(a, b);
    const int n = items_of(a, s);
    int64_t sum = 0;
    for (int k = 0; k < min(n, kFew); ++k) sum += item_units(a, s, k);
    pref[b] = n > kFew ? -1 : sum * a.cache.heads_kv;
  }
  __syncthreads();
  for (int b = warp; b < batch; b += blockDim.x >> 5) {
    if (pref[b] != -1) continue;
    const Sequence s = load_sequence(a, b);
    const int n = items_of(a, s);
    int64_t sum = 0;
    for (int k = lane; k < n; k += 32) sum += item_units(a, s, k);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncwarp();
    if (lane == 0) pref[b] = sum * a.cache.heads_kv;
  }
  __syncthreads();
  if (warp == 0) {
    // Exclusive prefix sums in place; pref[batch] is the total.
    int64_t run = 0;
    for (int b0 = 0; b0 < batch; b0 += 32) {
      const int64_t own = b0 + lane < batch ? pref[b0 + lane] : 0;
      int64_t incl = own;
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (b0 + lane < batch) pref[b0 + lane] = run + incl - own;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    __syncwarp();
    const int64_t total = run;
    const int64_t g0 = total * blockIdx.x / gridDim.x;
    const int64_t g1 = total * (blockIdx.x + 1) / gridDim.x;
    if (g1 > g0) {
      // The largest b with pref[b] <= g0 (sequences without rows share their successor's start).
      int lo = 0, hi = batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pref[mid] <= g0) lo = mid;
        else hi = mid - 1;
      }
      const Sequence s = load_sequence(a, lo);
      const int64_t own = (lo + 1 < batch ? pref[lo + 1] : total) - pref[lo];
      const int64_t per_head = own / a.cache.heads_kv;
      int64_t rem = g0 - pref[lo];
      const int hkv = static_cast<int>(rem / per_head);
      rem -= hkv * per_head;
      // The item that holds unit rem of this (sequence, head).
      const int n = items_of(a, s);
      int64_t before = 0;
      int k = 0;
      for (int k0 = 0; k0 < n; k0 += 32) {
        const int64_t u = k0 + lane < n ? item_units(a, s, k0 + lane) : 0;
        int64_t incl = u;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + incl > rem);
        if (past != 0) {
          const int at = __ffs(past) - 1;
          before += __shfl_sync(0xffffffffu, incl - u, at);
          k = k0 + at;
          break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) {
        sh->start[0] = lo;
        sh->start[1] = hkv;
        sh->start[2] = k;
        sh->start[3] = static_cast<int>(rem - before);
      }
    }
    if (lane == 0) sh->units = g1 - g0;
  }
}

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

// --------------------------------------------------------------------------------------------
// 8-bit codes
// --------------------------------------------------------------------------------------------

// Four codes as two pairs of exact bf16 or fp16 values. fp16: the byte 128 + q in the low bits of
// 1024 is 1152 + q. bf16: 128 + (q & 127), less 128 or (q negative) 256.
template <typename T>
__device__ __forceinline__ void codes_to_16bit(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if constexpr (std::is_same<T, __half>::value) {
    x ^= 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    lo = *reinterpret_cast<uint32_t*>(&r);
    r = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    hi = *reinterpret_cast<uint32_t*>(&r);
  } else {
    uint32_t y[2] = {__byte_perm(x, 0, 0x4140), __byte_perm(x, 0, 0x4342)};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t p = (y[i] & 0x007f007fu) | 0x43004300u, m = (y[i] & 0x00800080u) | 0x43004300u;
      __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&p),
                                 *reinterpret_cast<__nv_bfloat162*>(&m));
      (i == 0 ? lo : hi) = *reinterpret_cast<uint32_t*>(&r);
    }
  }
}

// A [128 x D] code tile to a 16-bit tile of 128-byte-swizzled [128 x 64] boxes, by 128 threads:
// 16 codes each per step. The lanes of columns 64-127 store their two chunks in the other order,
// which keeps the eight lanes of a store phase on different banks.
template <typename T, int D>
__device__ __forceinline__ void convert_tile(const uint8_t* codes, uint8_t* tile, int tid) {
  constexpr int kChunks = D / 16;
#pragma unroll 4
  for (int i = 0; i < kChunks; ++i) {
    const int at = i * 128 + tid;
    const int row = at / kChunks, c = at % kChunks;
    const uint4 x = *reinterpret_cast<const uint4*>(codes + at * 16);
    uint4 y[2];
    codes_to_16bit<T>(x.x, y[0].x, y[0].y);
    codes_to_16bit<T>(x.y, y[0].z, y[0].w);
    codes_to_16bit<T>(x.z, y[1].x, y[1].y);
    codes_to_16bit<T>(x.w, y[1].z, y[1].w);
    uint8_t* box = tile + (c >> 2) * kBoxBytes;
    const int chunk = (2 * c) & 7;
    const int swap = c >> 2;
    *reinterpret_cast<uint4*>(box + sw128_offset(row, chunk + swap)) = swap ? y[1] : y[0];
    *reinterpret_cast<uint4*>(box + sw128_offset(row, chunk + 1 - swap)) = swap ? y[0] : y[1];
  }
}

// --------------------------------------------------------------------------------------------
// Softmax
// --------------------------------------------------------------------------------------------

// 2^x of a row's 128 scores, row sums in ps, P packed to 16 bits in TMEM columns [0, 64) of the
// row's S region, published in two halves of 64 keys. x = s sl2 + nref (16-bit caches), or
// z + nref with the sum weighted by 1 / sv (int8: rsv).
template <typename P, bool kInt8>
__device__ __forceinline__ void exp_store(const float* sf, float sl2, float nref, const float* rsv,
                                          float (&ps)[4], uint32_t taddr_s, uint64_t* bars) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t pk[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      const int i = half * 64 + 2 * c;
      float x0, x1;
      if constexpr (kInt8) {
        fadd2(x0, x1, sf[i], sf[i + 1], nref, nref);
      } else {
        ffma2(x0, x1, sf[i], sf[i + 1], sl2, sl2, nref, nref);
      }
      const float p0 = ex2(x0), p1 = ex2(x1);
      const int acc = (c & 1) * 2;
      if constexpr (kInt8) {
        const float2 r = *reinterpret_cast<const float2*>(rsv + i);
        ffma2(ps[acc], ps[acc + 1], p0, p1, r.x, r.y, ps[acc], ps[acc + 1]);
      } else {
        fadd2(ps[acc], ps[acc + 1], ps[acc], ps[acc + 1], p0, p1);
      }
      pk[c] = pack2<P>(p0, p1);
    }
    tmem_st32(taddr_s + half * 32, pk);
    tmem_st_wait();
    tc_fence_before();
    mbar_arrive(&bars[half]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* x, float scale) {
  uint4 r;
  r.x = pack2<T>(x[0] * scale, x[1] * scale);
  r.y = pack2<T>(x[2] * scale, x[3] * scale);
  r.z = pack2<T>(x[4] * scale, x[5] * scale);
  r.w = pack2<T>(x[6] * scale, x[7] * scale);
  return r;
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
  using P = typename std::conditional<kInt8, __half, T>::type;   // weights, and V as multiplied
  using Sh = Shared<G::kSlots, G::kCodeSlots>;
  constexpr int kSlots = G::kSlots;
  constexpr int kTileBytes = G::kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* q_smem = smem;
  uint8_t* ring = smem + G::kRingOffset;
  Sh* sh = reinterpret_cast<Sh*>(smem + G::kTailOffset);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    sh->abort_flag = 0;
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh->kv_full[i], kInt8 ? 128 : 1);
      mbar_init(&sh->kv_empty[i], 1);
    }
    for (int i = 0; i < G::kCodeSlots; ++i) {
      mbar_init(&sh->code_full[i], 1);
      mbar_init(&sh->code_empty[i], 128);
    }
    for (int i = 0; i < kScaleSlots; ++i) mbar_init(&sh->scale_full[i], 128);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh->q_full[t], 1);
      mbar_init(&sh->q_free[t], 1);
      mbar_init(&sh->s_full[t], 1);
      mbar_init(&sh->p_half[t][0], kBM);
      mbar_init(&sh->p_half[t][1], kBM);
      mbar_init(&sh->o_full[t], 1);
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
  find_share(a, sh, reinterpret_cast<int64_t*>(ring));
  fence_proxy_async_shared();   // the ring was written here; TMA writes it next
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const WaitGuard guard{reinterpret_cast<volatile int*>(&sh->abort_flag), a.status};
  Walk walk;
  Segment s;

  // Barrier phases run on across segments: each role counts the completions it has waited for.
  if (warp == kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- TMA producer -------------------------------
    // Per segment: Q tile 0, K, Q tile 1, V, K, V, ... Lane i issues copy i of a tile (a part of
    // box_rows cache rows and, at 16 bits, one of the column boxes) from the block it read one
    // tile ahead.
    constexpr int kCols = kInt8 ? 1 : G::kBoxes;
    const int parts = kBN / a.box_rows;
    const bool issues = lane < parts * kCols;
    const int part = lane / kCols, col = lane % kCols;
    const bool paged = a.cache.block_tables != nullptr;
    const int page_size = a.cache.page_size;
    const int max_blocks = paged ? a.cache.max_seqlen / page_size : 0;
    const uint32_t q_bytes = static_cast<uint32_t>(a.group * a.tile_tokens * D * 2);
    int issued = 0;              // K/V tiles issued
    int q_loads[2] = {0, 0};
    bool ok = true;
    walk.start(a, sh);
    while (ok && walk.next(a, s)) {
      if (s.tiles == 0) continue;
      const int32_t* table = a.cache.block_tables + s.b * a.cache.bt_stride;
      auto block_of = [&](int tile) -> int {
        if (!paged) return s.b;
        const int page = (tile * kBN + part * a.box_rows) / page_size;
        const int blk = issues && page < max_blocks ? __ldg(table + page) : -1;
        return blk >= 0 && blk < a.cache.num_blocks ? blk : -1;   // -1 reads as zeros
      };
      auto load_q = [&](int t) -> bool {
        if (s.dual ? t == 1 : s.count[t] == 0) return true;
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
      int blk = block_of(s.t0);
      ok = __all_sync(0xffffffffu, load_q(0));
      for (int tile = s.t0; ok && tile < s.t1; ++tile) {
        const int next_blk = tile + 1 < s.t1 ? block_of(tile + 1) : 0;
        const int key = tile * kBN + part * a.box_rows;
        const int row = paged ? key % page_size : key;
        for (int kind = 0; ok && kind < 2; ++kind) {
          constexpr int kRing = kInt8 ? G::kCodeSlots : kSlots;
          const int slot = issued % kRing;
          uint64_t* empty = kInt8 ? &sh->code_empty[slot] : &sh->kv_empty[slot];
          uint64_t* full = kInt8 ? &sh->code_full[slot] : &sh->kv_full[slot];
          if (issued >= kRing) ok = mbar_wait(empty, ((issued / kRing) - 1) & 1, guard);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(full, kInt8 ? G::kCodeBytes : kTileBytes);
          __syncwarp();
          if (issues) {
            const TmaCoords& c = kind == 0 ? a.kc : a.vc;
            uint8_t* dst = kInt8 ? smem + G::kCodeOffset + slot * G::kCodeBytes + part * a.box_rows * D
                                 : ring + slot * kTileBytes + col * kBoxBytes + part * a.box_rows * 128;
            tma_load_4d(dst, kind == 0 ? &tmk : &tmv, full, col * 64, tma_c(c, 1, row, s.hkv, blk),
                        tma_c(c, 2, row, s.hkv, blk), tma_c(c, 3, row, s.hkv, blk));
          }
          ++issued;
          if (tile == s.t0 && kind == 0) ok = __all_sync(0xffffffffu, load_q(1));
        }
        blk = next_blk;
      }
    }
    // Wait for the copies still landing before the CTA may exit.
    if (lane == 0) {
      constexpr int kRing = kInt8 ? G::kCodeSlots : kSlots;
      for (int t = 0; t < 2; ++t) {
        if (q_loads[t] > 0) mbar_wait(&sh->q_full[t], (q_loads[t] - 1) & 1, guard);
      }
      for (int i = issued > kRing ? issued - kRing : 0; i < issued; ++i) {
        uint64_t* full = kInt8 ? &sh->code_full[i % kRing] : &sh->kv_full[i % kRing];
        if (!mbar_wait(full, (i / kRing) & 1, guard)) break;
      }
    }
  } else if (warp == kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- MMA issuer -------------------------------
    // The warp runs this loop together; one lane issues every tcgen05.mma and commit. Key tile i
    // of a segment is ring entries 2 i (K) and 2 i + 1 (V). A one-tile item's second chain reads
    // Q tile 0 as well.
    constexpr int kFmtQk = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    constexpr int kFmtPv = std::is_same<P, __nv_bfloat16>::value ? 1 : 0;
    constexpr uint32_t kIdescQk = umma_idesc_f16(kFmtQk, kBM, kBN, 0);
    constexpr uint32_t kIdescPv = umma_idesc_f16(kFmtPv, kBM, D, 1);
    const bool leader = elect_one();
    const Desc q_desc(umma_smem_desc_sw128(smem_u32(q_smem), 16, 1024));
    const Desc ring_k(umma_smem_desc_sw128(smem_u32(ring), 16, 1024));
    const Desc ring_v(umma_smem_desc_sw128(smem_u32(ring), kBoxBytes, 1024));
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
    };
    int base = 0;                   // ring entry of the segment's first K tile
    int q_waits[2] = {0, 0}, p_waits[2] = {0, 0};
    bool ok = true, issued_any = false;
    auto wait_ring = [&](int i) {
      return __all_sync(0xffffffffu, mbar_wait(&sh->kv_full[i % kSlots], (i / kSlots) & 1, guard));
    };
    walk.start(a, sh);
    while (ok && walk.next(a, s)) {
      if (s.tiles == 0) continue;
      issued_any = true;
      const int steps = max(s.count[0], s.count[1]);
      // Q K^T of chain c's step j; frees what its last reader is.
      auto issue_qk = [&](int c, int j) -> bool {
        const int entry = base + 2 * s.place(c, j);
        if (!wait_ring(entry)) return false;
        tc_fence_after();
        const int slot = entry % kSlots;
        const int q_tile = s.dual ? 0 : c;
        if (leader) {
          const Desc qd = q_desc.at(q_tile * kTileBytes);
          const Desc kd = ring_k.at(slot * kTileBytes);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ss(tmem + c * 128, qd.at(kmajor_step(kk)).u64(), kd.at(kmajor_step(kk)).u64(),
                    kIdescQk, kk > 0);
          umma_commit(&sh->s_full[c]);
        }
        if (s.dual || c == 1) commit(&sh->kv_empty[slot]);
        // The chain's last Q K^T (of both chains for a shared Q tile: the one issued last).
        if (s.dual ? s.place(c, j) + 1 == s.t1 - s.t0 : j + 1 == s.count[c])
          commit(&sh->q_free[q_tile]);
        return true;
      };
      for (int c = 0; c < 2 && ok; ++c) {
        if (s.count[c] == 0) continue;
        if (!s.dual || c == 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&sh->q_full[c], q_waits[c] & 1, guard));
          if (!ok) break;
          ++q_waits[c];
        }
        ok = issue_qk(c, 0);
      }
      int zeroed = -1;              // last V entry whose rows past the length were zeroed
      for (int j = 0; j < steps && ok; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!ok) break;
          if (j < s.count[c]) {
            const int entry = base + 2 * s.place(c, j) + 1;
            const int slot = entry % kSlots;
            ok = wait_ring(entry);
            if (!ok) break;
            if constexpr (!kInt8) {
              const int keys = s.seq.len - s.tile(c, j) * kBN;   // of this tile
              if (keys < kBN && zeroed != entry) {
                zeroed = entry;
                uint8_t* v = ring + slot * kTileBytes;
                for (int i = lane; i < (kBN - keys) * 8 * G::kBoxes; i += 32) {
                  const int row = keys + i / (8 * G::kBoxes), chunk = i % (8 * G::kBoxes);
                  *reinterpret_cast<uint4*>(v + (chunk >> 3) * kBoxBytes + row * 128 +
                                            (chunk & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_shared();
                __syncwarp();
              }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = __all_sync(0xffffffffu, mbar_wait(&sh->p_half[c][half], p_waits[c] & 1, guard));
              if (!ok) break;
              tc_fence_after();
              if (leader) {
                const Desc vd = ring_v.at(slot * kTileBytes);
#pragma unroll
                for (int kq = 0; kq < kBN / 32; ++kq) {
                  const int kk = half * (kBN / 32) + kq;
                  umma_ts(tmem + 256 + c * 128, tmem + c * 128 + kk * 8,
                          vd.at(mnmajor_step(kk)).u64(), kIdescPv, (j > 0 || kk > 0) ? 1u : 0u);
                }
              }
            }
            if (!ok) break;
            ++p_waits[c];
            if (s.dual) commit(&sh->kv_empty[slot]);
          }
          // A two-tile item's V is read last by chain 1, whose tiles are the segment's.
          if (!s.dual && c == 1) commit(&sh->kv_empty[(base + 2 * j + 1) % kSlots]);
          if (j + 1 < s.count[c]) {
            ok = issue_qk(c, j + 1);
          } else if (j + 1 == s.count[c]) {
            commit(&sh->o_full[c]);
          }
        }
      }
      base += 2 * (s.t1 - s.t0);
    }
    // Every MMA issued has completed before TMEM may be released.
    if (issued_any) {
      commit(&sh->mma_done);
      mbar_wait(&sh->mma_done, 0, guard);
    }
  } else if (warp < kProducerWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::kSoftmaxRegs));
    // ------------------------------- softmax warpgroups -------------------------------
    const int c = warp >> 2;                  // chain
    const int quarter = warp & 3;             // TMEM lane quarter this warp may access
    const int row = quarter * 32 + lane;      // of the tile
    const uint32_t lane_field = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t taddr_s = tmem + c * 128 + lane_field;
    const uint32_t taddr_o = tmem + 256 + c * 128 + lane_field;
    const float sl2 = a.scale_log2;
    const int row_token = row / a.group;
    const int row_head = row - row_token * a.group;
    int s_waits = 0, o_waits[2] = {0, 0}, joins = 0;
    int kv_base = 0;                          // key tiles of earlier segments (int8: scale slots)
    int segments = 0;
    int4 meta0 = make_int4(0, 0, 0, 0), meta1 = make_int4(0, 0, 0, 0);
    bool ok = true;
    walk.start(a, sh);
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
      const int count = s.count[c];

      float m_ref = -INFINITY;  // log2-domain reference point of this row
      float l_sum = 0.f;
      for (int j = 0; j < count; ++j) {
        if (!mbar_wait(&sh->s_full[c], s_waits & 1, guard)) {
          ok = false;
          break;
        }
        ++s_waits;
        if (!warp_ok) {   // whatever P holds stays in rows that nobody reads
          tc_fence_after();
          tc_fence_before();
          mbar_arrive(&sh->p_half[c][0]);
          mbar_arrive(&sh->p_half[c][1]);
          continue;
        }
        tc_fence_after();
        uint32_t sr[128];
        tmem_ld32(taddr_s + 0, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
        tmem_ld32(taddr_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
        tmem_ld32(taddr_s + 64, *reinterpret_cast<uint32_t(*)[32]>(&sr[64]));
        tmem_ld32(taddr_s + 96, *reinterpret_cast<uint32_t(*)[32]>(&sr[96]));
        tmem_ld_wait();
        float* sf = reinterpret_cast<float*>(sr);
        const int k0 = s.tile(c, j) * kBN;
        const float* scales = nullptr;
        if constexpr (kInt8) {
          // z = s mult + add.
          const int at = kv_base + s.place(c, j);
          if (!mbar_wait(&sh->scale_full[at % kScaleSlots], (at / kScaleSlots) & 1, guard)) {
            ok = false;
            break;
          }
          scales = reinterpret_cast<const float*>(smem + G::kScaleOffset) +
                   (at % kScaleSlots) * 3 * kBN;
#pragma unroll
          for (int i = 0; i < 128; i += 4) {
            const float4 mul = *reinterpret_cast<const float4*>(scales + i);
            const float4 add = *reinterpret_cast<const float4*>(scales + kBN + i);
            ffma2(sf[i], sf[i + 1], sf[i], sf[i + 1], mul.x, mul.y, add.x, add.y);
            ffma2(sf[i + 2], sf[i + 3], sf[i + 2], sf[i + 3], mul.z, mul.w, add.z, add.w);
          }
        }
        const bool masked = k0 + kBN > s.seq.len ||
                            (a.causal && k0 + kBN - 1 > offset + tile_first);
        if (masked) {
          const int visible = limit - k0;  // keys [k0, k0 + visible) are visible to this row
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
        const float mt = kInt8 ? mx : (mx == -INFINITY ? -INFINITY : mx * sl2);

        // The reference point moves only when the maximum passes it by more than 2^8.
        float m_new = m_ref;
        if (m_ref == -INFINITY || mt > m_ref + kRescaleThreshold) m_new = fmaxf(m_ref, mt);
        const bool rescale = (m_new != m_ref) && (m_ref != -INFINITY);
        const float factor = rescale ? ex2(m_ref - m_new) : 1.f;
        if (rescale) l_sum *= factor;
        m_ref = m_new;
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;
        if (__any_sync(0xffffffffu, rescale)) {
          // P V of the chain's previous step has completed (s_full covers it) and this step's waits
          // for the first half of P.
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
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
        exp_store<P, kInt8>(sf, sl2, -ref, scales + 2 * kBN, ps, taddr_s, sh->p_half[c]);
        l_sum += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      }
      if (!ok) break;
      kv_base += s.t1 - s.t0;

      // The end of the segment. Its O is read before this warpgroup publishes the next segment's
      // first P, which the first P V that overwrites O waits for.
      if (count > 0) {
        if (!mbar_wait(&sh->o_full[c], o_waits[c] & 1, guard)) break;
        ++o_waits[c];
      }
      float m_other = -INFINITY, l_other = 0.f;
      if (s.dual) {
        // Chain 1 hands its (m, l) to chain 0, which reads both O and writes the joint result.
        const uint32_t phase = joins++ & 1;
        if (c == 1) {
          sh->x_ml[row] = make_float2(m_ref, l_sum);
          tc_fence_before();
          mbar_arrive(&sh->x_ready);
          if (!mbar_wait(&sh->x_done, phase, guard)) break;
          tc_fence_after();
          continue;
        }
        if (!mbar_wait(&sh->x_ready, phase, guard)) break;
        const float2 ml = sh->x_ml[row];
        m_other = ml.x;
        l_other = ml.y;
      }
      tc_fence_after();
      const bool join = s.count[1] > 0 && s.dual;
      const float m = fmaxf(m_ref, m_other);
      const float ref = m == -INFINITY ? 0.f : m;
      float f0 = ex2(m_ref - ref), f1 = ex2(m_other - ref);
      if (!s.dual) f0 = 1.f;
      const float l = s.dual ? l_sum * f0 + l_other * f1 : l_sum;
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
            tmem_ld32(taddr_o + 128 + i * 32, ow);
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
      // Thread r also holds key r of the tile: its scales are read one tile ahead, its block two.
      // A tile's scales go to slot (tile % kScaleSlots) before its K tile is published. The slot is
      // free: the ring entries before this K tile were refilled, so P V of the tile kScaleSlots
      // earlier has run, which follows that tile's softmax.
      const int tid = threadIdx.x - kConvertWarp * 32;
      const bool paged = a.cache.block_tables != nullptr;
      const int page_size = a.cache.page_size;
      const int max_blocks = paged ? a.cache.max_seqlen / page_size : 0;
      int done = 0;   // code tiles converted
      bool ok = true;
      walk.start(a, sh);
      while (ok && walk.next(a, s)) {
        if (s.tiles == 0) continue;
        const int32_t* table = a.cache.block_tables + s.b * a.cache.bt_stride;
        auto block_of = [&](int tile) -> int {
          if (!paged) return s.b;
          const int page = (tile * kBN + tid) / page_size;
          const int blk = page < max_blocks ? __ldg(table + page) : -1;
          return blk < a.cache.num_blocks ? blk : -1;
        };
        auto scales_of = [&](int tile, int blk, float& sk, float& sv) {
          const int key = tile * kBN + tid;
          sk = 0.f;
          sv = kMinScale;
          if (key < s.seq.len && blk >= 0) {
            const int64_t r = paged ? key % page_size : key;
            sk = a.cache.ks[blk * a.cache.ks_stride[0] + r * a.cache.ks_stride[1] +
                            s.hkv * a.cache.ks_stride[2]];
            sv = a.cache.vs[blk * a.cache.vs_stride[0] + r * a.cache.vs_stride[1] +
                            s.hkv * a.cache.vs_stride[2]];
          }
        };
        float sk, sv, sk_next = 0.f, sv_next = 0.f;
        scales_of(s.t0, block_of(s.t0), sk, sv);
        int blk_next = block_of(s.t0 + 1);
        for (int tile = s.t0; ok && tile < s.t1; ++tile) {
          if (tile + 1 < s.t1) {
            scales_of(tile + 1, blk_next, sk_next, sv_next);
            blk_next = block_of(tile + 2);
          }
          for (int kind = 0; ok && kind < 2; ++kind) {
            const int code_slot = done % G::kCodeSlots, slot = done % kSlots;
            ok = mbar_wait(&sh->code_full[code_slot], (done / G::kCodeSlots) & 1, guard) &&
                 (done < kSlots || mbar_wait(&sh->kv_empty[slot], ((done / kSlots) - 1) & 1, guard));
            if (!ok) break;
            const uint8_t* codes = smem + G::kCodeOffset + code_slot * G::kCodeBytes;
            uint8_t* dst = ring + slot * kTileBytes;
            if (kind == 0) {
              float* out = reinterpret_cast<float*>(smem + G::kScaleOffset) +
                           ((done / 2) % kScaleSlots) * 3 * kBN + tid;
              // Keys past the length have no weight. A scale that is not finite makes z, and so the
              // weight, not finite for the rows that see the key, and adds nothing to others' sums.
              const bool in = tile * kBN + tid < s.seq.len;
              sv = sv < kMinScale ? kMinScale : sv;
              out[0] = in ? sk * a.scale_log2 : 0.f;
              out[kBN] = in ? __log2f(sv) : -INFINITY;
              out[2 * kBN] = in && sv <= 0x1p+127f ? 1.f / sv : 0.f;
              mbar_arrive(&sh->scale_full[(done / 2) % kScaleSlots]);
              convert_tile<T, D>(codes, dst, tid);
            } else {
              convert_tile<__half, D>(codes, dst, tid);
            }
            fence_proxy_async_shared();
            mbar_arrive(&sh->kv_full[slot]);
            mbar_arrive(&sh->code_empty[code_slot]);
            ++done;
          }
          sk = sk_next;
          sv = sv_next;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::kOtherRegs));
    // ------------------------------- warps 10 and 11 -------------------------------
    // Rows of no sequence (before the first offset, behind the last) give 0 and -inf.
    const Ragged& r = a.ragged;
    int begin = 0, end = 0;
    if (r.cu != nullptr) {
      begin = min(max(__ldg(r.cu), 0), r.rows);
      end = min(max(__ldg(r.cu + r.batch), begin), r.rows);
    } else {
      end = static_cast<int>(min(static_cast<int64_t>(r.batch) * r.rows_per_seq,
                                 static_cast<int64_t>(r.rows)));
    }
    const int64_t missing = static_cast<int64_t>(begin + r.rows - end) * a.heads;
    for (int64_t i = blockIdx.x * 2 + warp - 10; i < missing; i += gridDim.x * 2) {
      const int64_t at = i / a.heads;
      const int head = static_cast<int>(i - at * a.heads);
      const int64_t out_row = at < begin ? at : end + (at - begin);
      T* orow = static_cast<T*>(a.o) + out_row * a.o_stride[0] + head * a.o_stride[1];
      if (lane < D / 8) reinterpret_cast<uint4*>(orow)[lane] = make_uint4(0, 0, 0, 0);
      if (lane == 0) a.lse[out_row * a.heads + head] = -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kProducerWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the partials of the items that were cut. Block (c, y) handles the item that CTA c opened
// without closing, if there is one: its parts are that slot and the first slots of the following
// CTAs, up to the one that closes it, combined in that order (CTAs whose share held no whole key
// tile of the item left none). A thread owns 8 columns of one row.
template <typename T, int D>
__global__ void __launch_bounds__(256) extend_merge_kernel(const __grid_constant__ ExtendArgs a,
                                                           int ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ int first_flags[kMaxCtas];   // flags of the CTAs' first slots
  const int cta = blockIdx.x;
  int open = -1;
  int4 meta = make_int4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int4 m = a.part_meta[2 * cta + i];
    if ((m.x & (kPartValid | kPartOpens | kPartCloses)) == (kPartValid | kPartOpens)) {
      open = 2 * cta + i;
      meta = m;
    }
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
  constexpr int kBatch = 4;   // parts whose loads are issued together
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
        m = m_new;
        l = l * keep + ml[i].y * f;
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
  constexpr int kSmem = G::kTailOffset + static_cast<int>(sizeof(Shared<G::kSlots, G::kCodeSlots>)) +
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
  if (int st = check_cuda(cudaGetLastError(), "extend_kernel launch")) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, (a.part_rows * (D / 8) + 255) / 256);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, extend_merge_kernel<T, D>, a, ctas),
                    "extend_merge_kernel launch");
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
  const int ps = c->page_size;
  if (c->block_tables != nullptr && !(ps == 8 || ps == 16 || ps == 32 || ps % 64 == 0))
    return fail(FLB_ERR_UNSUPPORTED, "paged cache: page_size %d must be 8, 16, 32 or a multiple of 64",
                ps);
  if (c->batch > kMaxBatch)
    return fail(FLB_ERR_UNSUPPORTED, "more than %d sequences in one call", kMaxBatch);
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

extern "C" size_t flb_extend_workspace_bytes(int32_t rows, int32_t heads, int32_t heads_kv,
                                             int32_t head_dim, int32_t sm_count) {
  if (rows <= 0 || heads <= 0 || heads_kv <= 0 || heads % heads_kv != 0 ||
      heads / heads_kv > kBM || head_dim <= 0 || sm_count <= 0)
    return 0;
  const size_t slots = 2 * static_cast<size_t>(sm_count);
  const size_t part = static_cast<size_t>(part_rows(rows, heads / heads_kv));
  return align256(slots * sizeof(int4)) + align256(slots * part * 2 * sizeof(float)) +
         slots * part * head_dim * sizeof(float);
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
  a.tile_tokens = kBM / a.group;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->softmax_scale) * 1.4426950408889634);
  a.cache = kv_view(c);
  const size_t slots = 2 * static_cast<size_t>(sm_count);
  a.part_rows = part_rows(p->rows, a.group);
  char* ws = static_cast<char*>(p->workspace);
  a.part_meta = reinterpret_cast<int4*>(ws);
  ws += align256(slots * sizeof(int4));
  a.part_ml = reinterpret_cast<float*>(ws);
  ws += align256(slots * static_cast<size_t>(a.part_rows) * 2 * sizeof(float));
  a.part_o = reinterpret_cast<float*>(ws);

  // Boxes of the cache: whole tiles of a contiguous cache, else rows that never cross a page.
  const int ps = c->page_size;
  a.box_rows = c->block_tables == nullptr || ps % kBN == 0 ? kBN : std::min(ps, 64);
  CUtensorMap tmq, tmk, tmv;
  const View4 kv = kv_view4(c, false), vv = kv_view4(c, true);
  if (c->dtype == FLB_INT8) {
    if (int st = encode_rows_map(&tmk, &a.kc, kv, a.box_rows, c->head_dim, FLB_INT8, false))
      return st;
    if (int st = encode_rows_map(&tmv, &a.vc, vv, a.box_rows, c->head_dim, FLB_INT8, false))
      return st;
  } else {
    if (int st = encode_rows_x64_map(&tmk, &a.kc, kv, a.box_rows, c->dtype)) return st;
    if (int st = encode_rows_x64_map(&tmv, &a.vc, vv, a.box_rows, c->dtype)) return st;
  }
  if (int st = encode_group_map(&tmq, p->q, p->rows, c->heads_kv, a.group, c->head_dim,
                                p->q_row_stride, p->q_head_stride, a.tile_tokens, p->dtype))
    return st;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (p->dtype == FLB_BF16)
    return launch_t<__nv_bfloat16>(c, a, tmq, tmk, tmv, sm_count, dev, stream);
  return launch_t<__half>(c, a, tmq, tmk, tmv, sm_count, dev, stream);
}
