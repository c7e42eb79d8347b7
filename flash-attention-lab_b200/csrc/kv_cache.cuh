// What the kernels of kv_cache.cu and extend.cu share: the device view of a KV cache and the map
// from a ragged row to its sequence, and (host) the argument checks of flb_kv_cache.
#pragma once

#include <cstdint>

#include "host_common.h"

namespace flb {

// Division of 0 <= n < 2^31 by a constant d >= 1: with 2^(shift - 1) < d <= 2^shift and
// mul = floor(2^32 (2^shift - d) / d) + 1, n / d = (n + (n mul >> 32)) >> shift.
struct FastDiv {
  uint32_t mul;
  int shift, d;

  static FastDiv of(int d) {
    FastDiv f{0, 0, d};
    while ((int64_t{1} << f.shift) < d) ++f.shift;
    f.mul = static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << f.shift) - d)) / d + 1);
    return f;
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((static_cast<uint32_t>(n) + __umulhi(static_cast<uint32_t>(n), mul)) >>
                            shift);
  }
};

// Keys per sequence: positions of the tile behind the last key stay in 31 bits.
constexpr int kMaxSeqlen = 1 << 30;

// A KV cache as the kernels see it. Strides in elements of the cache (or of the scales).
struct KvView {
  void* k;
  void* v;
  int64_t k_stride[3], v_stride[3];   // sequence or block, row, head
  float* ks;
  float* vs;
  int64_t ks_stride[3], vs_stride[3];
  const int32_t* block_tables;        // null: contiguous
  int64_t bt_stride;
  FastDiv page;                       // page_size (1 when contiguous)
  int num_blocks, max_blocks, max_seqlen, heads_kv, batch;

  // The (outer, row) of key `pos` of sequence b; false when it lies outside the cache.
  __device__ __forceinline__ bool locate(int b, int pos, int64_t& outer, int64_t& row) const {
    if (pos < 0 || pos >= max_seqlen) return false;
    outer = b;
    row = pos;
    if (block_tables != nullptr) {
      const int p = page.div(pos);
      const int blk = __ldg(block_tables + b * bt_stride + p);
      if (blk < 0 || blk >= num_blocks) return false;
      outer = blk;
      row = pos - p * page.d;
    }
    return true;
  }
};

// Ragged rows: sequence b owns rows [cu[b], cu[b + 1]), or rows_per_seq rows each (cu null).
struct Ragged {
  const int32_t* cu;
  int rows, rows_per_seq, batch;
};

// Where row t of a ragged call lives: the sequence b that owns it, its place in the sequence and
// the sequence's row count, of the rows that there are; false if no sequence owns it. Lane i of a warp asks for row t0 + i.
// cu is searched 32 ways at once for t0 (one dependent load per factor of 32 of the batch), and
// from there each lane steps to its own row's sequence.
__device__ __forceinline__ bool find_sequences(const Ragged& r, int t0, int lane, int& b, int& place,
                                               int& count) {
  const int t = t0 + lane;
  if (r.cu == nullptr) {
    b = t / r.rows_per_seq;
    const int start = b * r.rows_per_seq;   // at most t
    place = t - start;
    count = min(r.rows_per_seq, r.rows - start);
    return t < r.rows && b < r.batch;
  }
  int lo = 0, hi = r.batch;   // the largest b in [lo, hi) with cu[b] <= t0, or 0
  while (true) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const bool below = i < hi && __ldg(r.cu + i) <= t0;
    const int n = max(__popc(__ballot_sync(0xffffffffu, below)), 1);
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
    if (step == 1) break;
  }
  b = lo;
  int first = __ldg(r.cu + b), end = __ldg(r.cu + b + 1);
  while (t < r.rows && end <= t && b + 1 < r.batch) {
    ++b;
    first = end;
    end = __ldg(r.cu + b + 1);
  }
  first = max(first, 0);
  end = min(end, r.rows);
  place = t - first;
  count = end - first;
  return first <= t && t < end;
}

// Checks of an flb_kv_cache that do not depend on who uses it: required pointers, positive sizes,
// the dtype and its scales, head_dim 64 or 128, a consistent paged layout and 16-byte aligned rows.
int validate_kv_cache(const flb_kv_cache* c);
KvView kv_view(const flb_kv_cache* c);
// The [outer, rows, H_kv, D] view of the K or V array (outer: sequences or blocks).
View4 kv_view4(const flb_kv_cache* c, bool v);

}  // namespace flb
