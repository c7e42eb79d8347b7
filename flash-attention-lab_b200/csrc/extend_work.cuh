// What the kernels of extend.cu and extend_few.cu share: their arguments, how the work of a call
// is cut into shares, the 8-bit codes as 16-bit values, and rows of no sequence.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "extend_steps.h"
#include "kv_cache.cuh"
#include "sm100.cuh"

namespace flb {

constexpr int kBN = 128;              // keys per tile
constexpr float kRescaleThreshold = 8.0f;   // log2 units: weights stay <= 2^8
constexpr int kItemUnits = 2;         // fixed cost of an item, in halves of a two-tile key tile
constexpr int kMaxBatch = 16384;      // the units' prefix sums use the K/V ring before it fills
constexpr float kMinScale = 0x1p-100f;
constexpr float kMaxScale = 0x1p+127f;   // V scales above it make the rows that see their key NaN
constexpr int kMaxCtas = 256;         // SMs of a device (one CTA each)

struct ExtendArgs {
  void* o;
  float* lse;
  int64_t o_stride[2];                // row, head
  const int32_t* seq_lens;
  Ragged ragged;
  int* status;
  int heads, group, causal;
  int tile_tokens;                    // tokens per tile: (128, or 16 in extend_few.cu) / group
  FastDiv item_tokens;                // 2 tile_tokens
  int select;                         // kAllRows, or which sequences this launch takes:
  int few_tokens;                     // those of at most so many rows, or the others
  int wide_scales;                    // extend_few.cu: scales are read 16 bytes at a time
  int box_rows;                       // cache rows per TMA box (a box never crosses a page)
  float scale_log2;
  TmaCoords kc, vc;
  int k_once, v_once;                 // expanded dimensions of K and V (fold_expanded)
  // Partials: slot 2 c + i is CTA c's first (0) or last (1) item share. part_o holds
  // [slots][D / 8][part_rows][8], part_ml [slots][part_rows][2].
  int part_rows;
  float* part_o;
  float* part_ml;
  int4* part_meta;                    // [slots]: flags, first token's row, tokens, KV head
  KvView cache;
};

// A call over an int8 cache whose row counts are only known on the device runs both kernels: the one
// of extend_few.cu takes the sequences of at most few_tokens rows, the other one the rest.
enum : int { kAllRows = 0, kFewRows = 1, kManyRows = 2 };
constexpr int kFewTile = 16;          // most score rows of a sequence in extend_few.cu

enum : int { kPartValid = 1, kPartOpens = 2, kPartCloses = 4 };

__device__ __forceinline__ int tma_c(const TmaCoords& c, int slot, int s, int h, int b) {
  return c.pos_s == slot ? s : (c.pos_h == slot ? h : b);
}

// Caches may be expanded over sequences (or blocks) and KV heads: such a dimension of stride 0 has size 1
// in the tensor map, and its coordinate is 0 (or negative still: zeros).
enum : int { kOnceOuter = 1, kOnceHeads = 2 };
inline int fold_expanded(View4* v) {
  int once = 0;
  if (v->size[0] > 1 && v->stride[0] == 0) {
    v->size[0] = 1;
    once |= kOnceOuter;
  }
  if (v->size[2] > 1 && v->stride[2] == 0) {
    v->size[2] = 1;
    once |= kOnceHeads;
  }
  return once;
}
__device__ __forceinline__ int coordinate(int x, int once) { return once ? min(x, 0) : x; }

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
  if (a.select != kAllRows && (s.n <= a.few_tokens) != (a.select == kFewRows)) s.n = 0;
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
  return a.item_tokens.div(s.n + a.item_tokens.d - 1);
}
__device__ __forceinline__ int item_units(const ExtendArgs& a, const Sequence& s, int k) {
  const int first = k * 2 * a.tile_tokens;
  const int last = min(first + 2 * a.tile_tokens, s.n);
  const int weight = last - first <= a.tile_tokens ? 1 : 2;
  return kItemUnits + weight * tiles_seen(a, s, last);
}

// A CTA's part of an item: key tiles [t0, t1) of all `tiles`. dual: the tokens fit in one tile.
struct Segment : Steps {
  Sequence seq;
  int b, hkv, first, tokens;   // sequence, KV head, first token in it, tokens
  int t0, t1, tiles;

  // Chain c's j-th key tile.
  __device__ __forceinline__ int tile(int c, int j) const { return t0 + place(c, j); }
};

// Where a CTA's share starts (unit `at` of item k of a sequence and KV head) and its length.
struct Share {
  int b, hkv, k, at;
  int64_t units;
};

// Walks a CTA's share segment by segment; every role walks the same sequence of segments.
struct Walk {
  Sequence seq;
  int b, hkv, k, at;
  int64_t left;

  __device__ __forceinline__ void start(const ExtendArgs& a, const Share& sh) {
    b = sh.b;
    hkv = sh.hkv;
    k = sh.k;
    at = sh.at;
    left = sh.units;
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
      const int from = min(at, total);
      const int to = static_cast<int>(min(static_cast<int64_t>(total), at + left));
      s.t0 = (max(from - kItemUnits, 0) + weight - 1) / weight;
      s.t1 = (max(to - kItemUnits, 0) + weight - 1) / weight;
      left -= to - from;
      at = to;
      if (to == total) {
        at = 0;
        if (++k >= items_of(a, seq)) {
          k = 0;
          if (left > 0) {
            do {   // some later sequence has rows, or the next head's first: units are left
              if (++b >= a.ragged.batch) {
                b = 0;
                if (++hkv >= a.cache.heads_kv) {   // offsets that decrease promise too many
                  left = 0;
                  break;
                }
              }
              seq = load_sequence(a, b);
            } while (seq.n == 0);
          }
        }
      }
      if (s.t1 > s.t0 || (s.tiles == 0 && from == 0)) {
        const int n = s.t1 - s.t0;
        if (s.dual) {
          s.count0 = (n + 1) / 2;
          s.count1 = n / 2;
        } else {
          s.count0 = min(max(tiles_seen(a, s.seq, s.first + a.tile_tokens), s.t0), s.t1) - s.t0;
          s.count1 = n;
        }
        return true;
      }
    }
    return false;
  }
};

// l 2^d, d <= 0, for a row sum l. Over an int8 cache the sum is in units of 2^M where M holds the log2 of
// a V scale, 2^-100 to 2^127: l can be 2^100 while M is far below the reference point it moves to, and
// 2^d alone would be 0.
__device__ __forceinline__ float scale_sum(float l, float d) {
  if (d > -100.f) return l * ex2(d);
  const float half = ex2(0.5f * d);
  return (l * half) * half;
}

// x / y for 0 <= x, 0 < y: 32-bit where both fit (a 64-bit division takes hundreds of clocks).
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  return ((x | y) >> 31) != 0 ? x / y
                              : static_cast<int64_t>(static_cast<uint32_t>(x) /
                                                     static_cast<uint32_t>(y));
}

// Inclusive prefix sum over the lanes.
__device__ __forceinline__ int prefix_sum(int x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += v;
  }
  return x;
}

// Units of a sequence's items of one KV head, by a whole warp.
__device__ __forceinline__ int sequence_units(const ExtendArgs& a, const Sequence& s, int lane) {
  const int n = items_of(a, s);
  int sum = 0;
  for (int k = lane; k < n; k += 32) sum += item_units(a, s, k);
  return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(sum)));
}

// The share's start: unit `rem` of sequence b and head hkv. One warp.
__device__ __forceinline__ void locate_unit(const ExtendArgs& a, Share* sh, int hkv, int b,
                                            const Sequence& s, int rem, int lane) {
  const int n = items_of(a, s);
  int before = 0, k = 0;
  for (int k0 = 0; n > 1 && k0 < n; k0 += 32) {
    const int u = k0 + lane < n ? item_units(a, s, k0 + lane) : 0;
    const int incl = prefix_sum(u, lane);
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
    sh->b = b;
    sh->hkv = hkv;
    sh->k = k;
    sh->at = max(rem - before, 0);
  }
}

// Units [g0, g1) of CTA c: shares differ by at most one unit.
__device__ __forceinline__ void share_bounds(int64_t total, int64_t& g0, int64_t& g1) {
  const int64_t ctas = gridDim.x, c = blockIdx.x;
  const int64_t each = divide(total, ctas), more = total - each * ctas;
  g0 = each * c + min(c, more);
  g1 = g0 + each + (c < more ? 1 : 0);
}

// The units of a call in the order (KV head, sequence, item, key tile): the CTAs that run together
// read about the same keys of several heads, which share DRAM pages in a [.., H_kv, D] cache.
// Those of one head fit in 31 bits (max_units bounds them on the host).
//
// Finds this CTA's share. All threads; `pref` is shared memory for batch values. It ends without a
// barrier. Up to 32 sequences are one warp's work (a lane per sequence), which the start of a
// short call waits for; more go through shared memory.
__device__ __forceinline__ void find_share(const ExtendArgs& a, Share* sh, int* pref) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int batch = a.ragged.batch;
  constexpr int kFew = 16;   // items one thread sums by itself
  int64_t g0, g1;
  if (batch <= 32) {
    if (warp != 0) return;
    Sequence s{0, 0, 0};
    if (lane < batch) s = load_sequence(a, lane);
    const int n = items_of(a, s);
    int own = 0;
    if (n <= kFew) {
      for (int k = 0; k < n; ++k) own += item_units(a, s, k);
    }
    auto sequence_of = [&](int b) {
      return Sequence{__shfl_sync(0xffffffffu, s.row0, b), __shfl_sync(0xffffffffu, s.n, b),
                      __shfl_sync(0xffffffffu, s.len, b)};
    };
    for (uint32_t long_ones = __ballot_sync(0xffffffffu, n > kFew); long_ones != 0;
         long_ones &= long_ones - 1) {
      const int b = __ffs(long_ones) - 1;
      const int sum = sequence_units(a, sequence_of(b), lane);
      if (lane == b) own = sum;
    }
    const int incl = prefix_sum(own, lane);
    const int total = __shfl_sync(0xffffffffu, incl, 31);   // of one head
    share_bounds(static_cast<int64_t>(total) * a.cache.heads_kv, g0, g1);
    if (g1 > g0) {
      const int hkv = static_cast<int>(divide(g0, total));
      const int rem = static_cast<int>(g0 - static_cast<int64_t>(hkv) * total);
      const int b = max(__ffs(__ballot_sync(0xffffffffu, incl > rem)) - 1, 0);
      locate_unit(a, sh, hkv, b, sequence_of(b), rem - __shfl_sync(0xffffffffu, incl - own, b),
                  lane);
    }
    if (lane == 0) sh->units = g1 - g0;
    return;
  }
  for (int b = threadIdx.x; b < batch; b += blockDim.x) {
    const Sequence s = load_sequence(a, b);
    const int n = items_of(a, s);
    int sum = 0;
    for (int k = 0; k < min(n, kFew); ++k) sum += item_units(a, s, k);
    pref[b] = n > kFew ? -1 : sum;
  }
  __syncthreads();
  for (int b = warp; b < batch; b += blockDim.x >> 5) {
    if (pref[b] != -1) continue;
    const int sum = sequence_units(a, load_sequence(a, b), lane);
    __syncwarp();
    if (lane == 0) pref[b] = sum;
  }
  __syncthreads();
  if (warp != 0) return;
  // Exclusive prefix sums in place.
  int total = 0;   // of one head
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int own = b0 + lane < batch ? pref[b0 + lane] : 0;
    const int incl = prefix_sum(own, lane);
    if (b0 + lane < batch) pref[b0 + lane] = total + incl - own;
    total += __shfl_sync(0xffffffffu, incl, 31);
  }
  __syncwarp();
  share_bounds(static_cast<int64_t>(total) * a.cache.heads_kv, g0, g1);
  if (g1 > g0) {
    const int hkv = static_cast<int>(divide(g0, total));
    const int rem = static_cast<int>(g0 - static_cast<int64_t>(hkv) * total);
    // The largest b with pref[b] <= rem (sequences without rows share their successor's start).
    int lo = 0, hi = batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pref[mid] <= rem) lo = mid;
      else hi = mid - 1;
    }
    locate_unit(a, sh, hkv, lo, load_sequence(a, lo), rem - pref[lo], lane);
  }
  if (lane == 0) sh->units = g1 - g0;
}

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

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* x, float scale) {
  uint4 r;
  r.x = pack2<T>(x[0] * scale, x[1] * scale);
  r.y = pack2<T>(x[2] * scale, x[3] * scale);
  r.z = pack2<T>(x[4] * scale, x[5] * scale);
  r.w = pack2<T>(x[6] * scale, x[7] * scale);
  return r;
}

// Rows of no sequence (before the first offset, behind the last) give 0 and -inf: worker `index` of
// `workers` warps takes its share of them.
template <typename T, int D>
__device__ __forceinline__ void zero_other_rows(const ExtendArgs& a, int index, int workers,
                                                int lane) {
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
  for (int64_t i = index; i < missing; i += workers) {
    const int64_t at = i / a.heads;
    const int head = static_cast<int>(i - at * a.heads);
    const int64_t out_row = at < begin ? at : end + (at - begin);
    T* orow = static_cast<T*>(a.o) + out_row * a.o_stride[0] + head * a.o_stride[1];
    if (lane < D / 8) reinterpret_cast<uint4*>(orow)[lane] = make_uint4(0, 0, 0, 0);
    if (lane == 0) a.lse[out_row * a.heads + head] = -INFINITY;
  }
}

// Launches the kernel of extend_few.cu for an int8 cache (queries q, rows of 16 bits; a filled for
// its tile) with `ctas` CTAs.
int launch_extend_few(const ExtendArgs& a, const flb_kv_cache* c, const void* q,
                      int64_t q_row_stride, int64_t q_head_stride, int dtype, int ctas, int dev,
                      cudaStream_t stream);

}  // namespace flb
