// Attention of a few new rows per sequence over an int8 KV cache: single-token decode, and chunks
// whose (tokens x query heads of one KV head) are at most 16 score rows. Same operator, work split
// and partials as extend.cu; HBM bound (2 H_kv (D + 4) bytes per key), so the codes go from shared
// memory straight into the registers of 16 x 8 x 16 warp MMAs instead of through 16-bit tiles. One
// row of 8 sequences of 24K keys, 32 query and 8 KV heads, D 128 (415 MB): 80 us with the merge,
// 5.2 TB/s; the first tcgen05 form of extend.cu took 297 us. Roundings to fewer than 32 bits: bf16 queries
// to fp16 (below), the weights to fp16, the result to q's type.
//
//  * One CTA per SM: two warps stream [128 keys x D] tiles of K and of V codes by TMA, one turns the
//    keys' scales into what the scores need (below) beside them in the ring stage, and eight consumer
//    warps take 16 keys of a tile each, every warp with its own online softmax; their results are
//    joined in a fixed order at the end of a segment. (One producer warp for copies and scales, with
//    a table load per key, bounded 16-row pages: 5000 clocks per tile where the consumers took 2400.
//    Sixteen consumers in two groups on alternate tiles: 137 us against 129 with eight, whose issue
//    slots are 43 % used.)
//  * Keys are the M rows of the MMAs and score rows their N columns, in one or two blocks of 8: the
//    usual group of up to 8 heads costs half the MMAs, exponentials and registers of 16 score rows.
//  * Q is the B operand, in fp16: bf16 queries are scaled to [1, 2) of their row's maximum by a
//    power of two, which is exact down to 2^-17 of the maximum and off by at most 2^-25 of it
//    below. The order of a dot product is free, so thread t of a quad takes D / 4 consecutive values
//    of its keys' rows (16-byte shared loads) and the same ones of Q.
//  * V^T is the A operand of O^T = V^T P^T, by transposed 8 x 8 matrix loads of byte pairs: a
//    register then holds columns d and d + 1 of two keys, M rows g and g + 8 of the fragment. P
//    becomes the B operand by an 8 x 8 transpose in registers.
//  * The scales act as in extend.cu: z = s mult + log2 sv, w = 2^(z - M) in fp16. The row sum takes its
//    terms 2^(z - log2 sv - M) by an exponential of their own: w / sv would lose keys whose sv is 2^100
//    below the largest. (One row of 8 sequences of 16K-32K keys takes 83 us with either.)
#include <algorithm>

#include "extend_work.cuh"

namespace flb {
namespace {

constexpr int kWarps = kBN / 16;      // consumers: 16 keys of a tile each

// kBlocks: 8-row blocks of score rows (1 or 2).
template <int D, int kBlocks>
struct FewGeometry {
  static constexpr int kRows = 8 * kBlocks;
  static constexpr int kCopyWarp = kWarps;               // TMA of K, and kCopyWarp + 1 of V
  static constexpr int kScaleWarp = kWarps + 2;
  static constexpr int kThreads = (kWarps + 3) * 32;
  static constexpr int kTileBytes = kBN * D;             // K or V codes
  static constexpr int kStages = D == 128 ? 4 : 8;       // 128 KB of codes
  static constexpr int kScaleOffset = kStages * 2 * kTileBytes;
  static constexpr int kScaleBytes = 2 * kBN * 4;        // sk and log2 sv of one stage
  static constexpr int kRawTiles = 8;                    // scales as read: see the scale warp
  static constexpr int kRawOffset = kScaleOffset + kStages * kScaleBytes;
  static constexpr int kJoinOffset = kRawOffset + kRawTiles * 2 * kBN * 4;
  static constexpr int kJoinBytes = kWarps * kRows * (D + 2) * 4;
  static constexpr int kTailOffset = kJoinOffset + kJoinBytes;
  static_assert(kMaxBatch * 4 <= kScaleOffset, "prefix sums fit in the ring");
};

template <int kStages>
struct FewShared {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  int abort_flag;
  Share share;
};

// Copies 16 or 4 bytes to shared memory (the shorter form: zeros unless valid).
__device__ __forceinline__ void cp_async_16(uint32_t dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 4 : 0)
               : "memory");
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The block table of one sequence as a warp reads it: 32 entries from `base` and the 32 after
// them, one per lane, the second half a window ahead. Pages are asked for in tile order; a tile's
// lie in [base, base + 64) once advance() was called with its first one.
struct BlockWindow {
  const int32_t* table;
  int base, cur, next;

  __device__ __forceinline__ int entry(const KvView& c, int page) const {
    const int blk = page < c.max_blocks ? __ldg(table + page) : -1;
    return blk >= 0 && blk < c.num_blocks ? blk : -1;   // -1 reads as zeros
  }
  __device__ __forceinline__ void start(const KvView& c, int b, int first_page, int lane) {
    table = c.block_tables + b * c.bt_stride;
    base = first_page;
    cur = entry(c, base + lane);
    next = entry(c, base + 32 + lane);
  }
  __device__ __forceinline__ void advance(const KvView& c, int first_page, int lane) {
    if (first_page >= base + 32) {
      base += 32;
      cur = next;
      next = entry(c, base + 32 + lane);
    }
  }
  __device__ __forceinline__ int at(int page) const {   // every lane calls this
    const int i = page - base;
    const int lo = __shfl_sync(0xffffffffu, cur, i & 31);
    const int hi = __shfl_sync(0xffffffffu, next, i & 31);
    return i < 32 ? lo : hi;
  }
};

// Byte offset of 16-byte chunk c of row r in a code tile as TMA wrote it (128- or 64-byte swizzle).
template <int D>
__device__ __forceinline__ uint32_t code_offset(uint32_t r, uint32_t c) {
  return D == 128 ? sw128_offset(r, c) : r * 64u + ((c ^ ((r >> 1) & 3u)) << 4);
}

// Bytes 0, 2 and 1, 3 of a register of codes as two pairs of fp16 (see codes_to_16bit).
__device__ __forceinline__ void code_columns(uint32_t x, uint32_t& even, uint32_t& odd) {
  x ^= 0x80808080u;
  const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  uint32_t a = __byte_perm(x, 0x64646464u, 0x4240), b = __byte_perm(x, 0x64646464u, 0x4341);
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
  even = *reinterpret_cast<uint32_t*>(&r);
  r = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
  odd = *reinterpret_cast<uint32_t*>(&r);
}

// The 8 x 8 matrix of 16-bit values that a warp holds (row lane / 4, columns 2 (lane % 4) + {0, 1}),
// transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// True on all kThreads consumer threads when pred holds on any of them.
template <int kThreads>
__device__ __forceinline__ bool consumers_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "n"(kThreads)
      : "memory");
  return r != 0;
}

struct QueryView {
  const void* q;
  int64_t stride[2];   // row, head
};

template <typename T, int D, int kBlocks>
__global__ void __launch_bounds__(FewGeometry<D, kBlocks>::kThreads, 1)
    extend_few_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ QueryView qv,
                      const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using G = FewGeometry<D, kBlocks>;
  constexpr int kStages = G::kStages;
  constexpr int kRows = G::kRows;
  constexpr int kSteps = D / 16;    // MMA steps over head_dim, and 16-column chunks of V
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  auto* sh = reinterpret_cast<FewShared<kStages>*>(smem + G::kTailOffset);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (warp == G::kScaleWarp && lane == 0) {   // warp 0 finds the share
    sh->abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh->full[i], 34);   // the bytes of K and of V, and each lane's scales
      mbar_init(&sh->empty[i], kWarps);
    }
    fence_barrier_init();
  }
  if (warp == G::kCopyWarp && lane == 0) {
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  find_share(a, &sh->share, reinterpret_cast<int*>(smem));
  fence_proxy_async_shared();   // the ring was written here; TMA writes it next
  __syncthreads();
  const WaitGuard guard{reinterpret_cast<volatile int*>(&sh->abort_flag), a.status};
  Walk walk;
  Segment s{};
  walk.start(a, sh->share);

  if (warp < G::kScaleWarp && warp >= G::kCopyWarp) {
    // ------------------------------- copies -------------------------------
    // Lane i issues copy i of a tile, a part of box_rows rows. Small pages are many copies, whose
    // issue one warp for K and V could not keep up with (16-row pages: 2000 clocks per tile).
    const bool is_v = warp != G::kCopyWarp;
    const int offset = lane * a.box_rows;   // of the part's keys
    const bool issues = offset < kBN;
    const bool paged = a.cache.block_tables != nullptr;
    const CUtensorMap* map = is_v ? &tmv : &tmk;
    const TmaCoords& c = is_v ? a.vc : a.kc;
    const int once = is_v ? a.v_once : a.k_once;
    BlockWindow window;
    int issued = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      if (paged) window.start(a.cache, s.b, a.cache.page.div(s.t0 * kBN), lane);
      for (int tile = s.t0; tile < s.t1; ++tile) {
        const int key = tile * kBN + offset;
        int blk = s.b, row = key;
        if (paged) {
          const int page = a.cache.page.div(key);
          window.advance(a.cache, __shfl_sync(0xffffffffu, page, 0), lane);
          blk = window.at(issues ? page : window.base);
          row = key - page * a.cache.page.d;
        }
        const int st = issued % kStages;
        ok = issued < kStages || mbar_wait(&sh->empty[st], ((issued / kStages) - 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sh->full[st], G::kTileBytes);
        __syncwarp();
        if (issues) {
          const int h = coordinate(s.hkv, once & kOnceHeads), at = coordinate(blk, once & kOnceOuter);
          tma_load_4d(smem + (2 * st + (is_v ? 1 : 0)) * G::kTileBytes + offset * D, map,
                      &sh->full[st], 0, tma_c(c, 1, row, h, at), tma_c(c, 2, row, h, at),
                      tma_c(c, 3, row, h, at));
        }
        ++issued;
      }
    }
    // Wait for the copies still landing before the CTA may exit.
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
      if (!mbar_wait(&sh->full[i % kStages], (i / kStages) & 1, guard)) break;
    }
    return;
  }
  if (warp == G::kScaleWarp) {
    // ------------------------------- scales -------------------------------
    // Lane i turns the scales of keys 4 i .. 4 i + 3 of a tile into sk and log2 sv. They lie
    // in one page, as 16 contiguous bytes with a.wide_scales. They are copied to shared memory
    // kRawTiles - 1 tiles ahead, each lane its own: a warp alone runs about 5 clocks per instruction
    // and cannot wait for memory in every tile (registers one tile ahead: 2200 clocks per
    // tile, where the consumers take 950).
    constexpr int kRawTiles = G::kRawTiles;
    const bool paged = a.cache.block_tables != nullptr;
    const int64_t ks_row = a.cache.ks_stride[1], vs_row = a.cache.vs_stride[1];
    const uint32_t raw = smem_u32(smem + G::kRawOffset) + lane * 16;
    BlockWindow window;
    int issued = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      if (paged) window.start(a.cache, s.b, a.cache.page.div(s.t0 * kBN), lane);
      const float* ks = a.cache.ks + s.hkv * a.cache.ks_stride[2];
      const float* vs = a.cache.vs + s.hkv * a.cache.vs_stride[2];
      if (!paged) {
        ks += s.b * a.cache.ks_stride[0];
        vs += s.b * a.cache.vs_stride[0];
      }
      // Keys past the length are not read: they stay hidden, whatever their scales.
      auto fetch = [&](int tile) {
        if (tile < s.t1) {
          const int key = tile * kBN + 4 * lane;
          const float *k = ks, *v = vs;
          int row = key, keys = s.seq.len - key;
          if (paged) {
            const int page = a.cache.page.div(key);
            window.advance(a.cache, __shfl_sync(0xffffffffu, page, 0), lane);
            const int blk = window.at(page);
            if (blk < 0) keys = 0;
            k += max(blk, 0) * a.cache.ks_stride[0];
            v += max(blk, 0) * a.cache.vs_stride[0];
            row = key - page * a.cache.page.d;
          }
          k += row * ks_row;
          v += row * vs_row;
          const uint32_t dst = raw + (tile - s.t0) % kRawTiles * (2 * kBN * 4);
          if (a.wide_scales && keys >= 4) {
            cp_async_16(dst, k);
            cp_async_16(dst + kBN * 4, v);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool in = i < keys;
              cp_async_4(dst + 4 * i, in ? k + i * ks_row : a.cache.ks, in);
              cp_async_4(dst + kBN * 4 + 4 * i, in ? v + i * vs_row : a.cache.vs, in);
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      for (int i = 0; i < kRawTiles - 1; ++i) fetch(s.t0 + i);
      for (int tile = s.t0; tile < s.t1; ++tile) {
        fetch(tile + kRawTiles - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kRawTiles - 1) : "memory");
        const float4* from = reinterpret_cast<const float4*>(
            smem + G::kRawOffset + (tile - s.t0) % kRawTiles * (2 * kBN * 4)) + lane;
        const float4 sk4 = from[0];
        const float4 sv4 = from[kBN / 4];
        float sk[4] = {sk4.x, sk4.y, sk4.z, sk4.w};
        const float sv[4] = {sv4.x, sv4.y, sv4.z, sv4.w};
        const int st = issued % kStages;
        ok = issued < kStages || mbar_wait(&sh->empty[st], ((issued / kStages) - 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float add[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // A V scale that is not finite makes the score NaN: it reaches the rows that see the key
          // and adds nothing to the sums of the others.
          const bool finite = sv[i] <= kMaxScale;
          if (!finite) sk[i] = __int_as_float(0x7fffffff);
          add[i] = finite ? lg2(fmaxf(sv[i], kMinScale)) : 0.f;
        }
        float4* dst = reinterpret_cast<float4*>(smem + G::kScaleOffset + st * G::kScaleBytes) + lane;
        dst[0] = make_float4(sk[0], sk[1], sk[2], sk[3]);
        dst[kBN / 4] = make_float4(add[0], add[1], add[2], add[3]);
        mbar_arrive(&sh->full[st]);
        ++issued;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    zero_other_rows<T, D>(a, blockIdx.x, gridDim.x, lane);
    return;
  }

  // ------------------------------- consumers -------------------------------
  const int g = lane >> 2;    // fragment row group
  const int t4 = lane & 3;    // thread in quad
  float* join_m = reinterpret_cast<float*>(smem + G::kJoinOffset);   // [warps][kRows]
  float* join_l = join_m + kWarps * kRows;
  float* join_o = join_l + kWarps * kRows;                           // [warps][kRows][D]
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t v_row = static_cast<uint32_t>(warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7));
  const uint32_t v_chunk = static_cast<uint32_t>(lane >> 4);
  int base = 0;               // tiles of earlier segments
  int segments = 0;
  int4 meta0 = make_int4(0, 0, 0, 0), meta1 = make_int4(0, 0, 0, 0);
  bool ok = true;
  while (walk.next(a, s)) {
    const bool first_segment = segments++ == 0;
    const int rows = s.tokens * a.group;
    // Q fragments: rows 8 nb + g, values [t4 D / 4, (t4 + 1) D / 4). Scores: this thread has rows
    // 8 nb + 2 t4 + {0, 1} of keys g and g + 8.
    uint32_t qb[kBlocks][kSteps][2];
    float row_scale[kBlocks][2];
    int limit[kBlocks][2];    // keys that the row sees
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
      const int row = 8 * nb + g;
      const int token = row / a.group, head = s.hkv * a.group + row - token * a.group;
      const uint2* src = reinterpret_cast<const uint2*>(
          static_cast<const T*>(qv.q) + (s.seq.row0 + s.first + token) * qv.stride[0] +
          head * qv.stride[1] + t4 * (D / 4));
      uint2 x[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) x[k] = row < rows ? __ldg(src + k) : make_uint2(0, 0);
      float up = a.scale_log2;
      if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qb[nb][k][0] = x[k].x;
          qb[nb][k][1] = x[k].y;
        }
      } else {
        // The exponent of the row's maximum (magnitudes compare as integers).
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          top = max(top, max(x[k].x & 0x7fffu, (x[k].x >> 16) & 0x7fffu));
          top = max(top, max(x[k].y & 0x7fffu, (x[k].y >> 16) & 0x7fffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max(static_cast<int>(top >> 7), 1), 253);
        const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        up *= __uint_as_float(static_cast<uint32_t>(e) << 23);
        auto half_pair = [&](uint32_t v) {
          return pack2<__half>(__uint_as_float(v << 16) * down,
                               __uint_as_float(v & 0xffff0000u) * down);
        };
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qb[nb][k][0] = half_pair(x[k].x);
          qb[nb][k][1] = half_pair(x[k].y);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[nb][e] = __shfl_sync(0xffffffffu, up, (2 * t4 + e) * 4);
        limit[nb][e] = a.causal ? min(s.seq.len, s.seq.len - s.seq.n + s.first +
                                                     (8 * nb + 2 * t4 + e) / a.group + 1)
                                : s.seq.len;
      }
    }
    // O^T: columns 16 c + 2 g (elements 0, 1) and 16 c + 2 g + 1 (2, 3) of rows 8 nb + 2 t4 + {0, 1}.
    float o[kBlocks][kSteps][4];
    float m_ref[kBlocks][2], l_sum[kBlocks][2];   // log2-domain reference point; share of the sum
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        o[nb][c][0] = o[nb][c][1] = o[nb][c][2] = o[nb][c][3] = 0.f;
      m_ref[nb][0] = m_ref[nb][1] = -INFINITY;
      l_sum[nb][0] = l_sum[nb][1] = 0.f;
    }

    for (int tile = s.t0; tile < s.t1; ++tile) {
      const int pos = base + tile - s.t0, st = pos % kStages;
      ok = mbar_wait(&sh->full[st], (pos / kStages) & 1, guard);
      if (!ok) break;
      const uint8_t* kt = smem + 2 * st * G::kTileBytes;
      const uint32_t vt = smem_base + (2 * st + 1) * G::kTileBytes;
      const float* scales = reinterpret_cast<const float*>(smem + G::kScaleOffset +
                                                           st * G::kScaleBytes) + warp * 16 + g;
      const int key = tile * kBN + warp * 16 + g;   // and key + 8

      // Two accumulators per block: a chain of D / 16 dependent MMAs is half as long.
      float z[kBlocks][4], y[kBlocks][4];
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) z[nb][e] = y[nb][e] = 0.f;
      }
      {
        uint4 x[2][D / 64];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int i = 0; i < D / 64; ++i)
            x[r][i] = *reinterpret_cast<const uint4*>(
                kt + code_offset<D>(warp * 16 + 8 * r + g, t4 * (D / 64) + i));
        }
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t word0[4] = {x[0][i].x, x[0][i].y, x[0][i].z, x[0][i].w};
          const uint32_t word1[4] = {x[1][i].x, x[1][i].y, x[1][i].z, x[1][i].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t ka[4];
            codes_to_16bit<__half>(word0[w], ka[0], ka[2]);
            codes_to_16bit<__half>(word1[w], ka[1], ka[3]);
#pragma unroll
            for (int nb = 0; nb < kBlocks; ++nb)
              mma_16816<__half>((w & 1) ? y[nb] : z[nb], ka, qb[nb][4 * i + w][0],
                                qb[nb][4 * i + w][1]);
          }
        }
      }
      const float sk[2] = {scales[0], scales[8]};
      const float add[2] = {scales[kBN], scales[kBN + 8]};
      // Element e: row e & 1, key g + 8 (e >> 1). The reference point moves only when a score
      // passes it by more than 2^8, and the warp's maximum is taken only then.
      bool above = false;
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e & 1, k = e >> 1;
          const float v = fmaf((z[nb][e] + y[nb][e]) * row_scale[nb][r], sk[k], add[k]);
          z[nb][e] = key + 8 * k < limit[nb][r] ? v : -INFINITY;
          above |= z[nb][e] > m_ref[nb][r] + kRescaleThreshold;
        }
      }
      if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(z[nb][r], z[nb][2 + r]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (mx > m_ref[nb][r] + kRescaleThreshold) {
              const float factor = ex2(m_ref[nb][r] - mx);   // 0 for the first keys
              l_sum[nb][r] = scale_sum(l_sum[nb][r], m_ref[nb][r] - mx);
              m_ref[nb][r] = mx;
#pragma unroll
              for (int c = 0; c < kSteps; ++c) {
                o[nb][c][r] *= factor;
                o[nb][c][2 + r] *= factor;
              }
            }
          }
        }
      }
      uint32_t pb[kBlocks][2];
#pragma unroll
      for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e & 1;
          const float ref = m_ref[nb][r] == -INFINITY ? 0.f : m_ref[nb][r];
          const float x = z[nb][e] - ref;
          z[nb][e] = ex2(x);
          // The square of a root: the term may be below the exponential's range, 2^-126.
          const float root = ex2(fmaf(x, 0.5f, -0.5f * add[e >> 1]));
          l_sum[nb][r] = fmaf(root, root, l_sum[nb][r]);
        }
        pb[nb][0] = transpose8x8(pack2<__half>(z[nb][0], z[nb][1]));
        pb[nb][1] = transpose8x8(pack2<__half>(z[nb][2], z[nb][3]));
      }
#pragma unroll
      for (int c = 0; c < kSteps; c += 2) {
        uint32_t v[4];   // keys 0-7 and 8-15 of chunk c, then of chunk c + 1
        ldsm_x4_trans(vt + code_offset<D>(v_row, c + v_chunk), v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t va[4];
          code_columns(v[2 * i], va[0], va[1]);
          code_columns(v[2 * i + 1], va[2], va[3]);
#pragma unroll
          for (int nb = 0; nb < kBlocks; ++nb)
            mma_16816<__half>(o[nb][c + i], va, pb[nb][0], pb[nb][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->empty[st]);
    }
    base += s.t1 - s.t0;

    // Join the warps. Every consumer is past the previous segment's reads after the first barrier.
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l_sum[nb][r] += __shfl_xor_sync(0xffffffffu, l_sum[nb][r], 4);
        l_sum[nb][r] += __shfl_xor_sync(0xffffffffu, l_sum[nb][r], 8);
        l_sum[nb][r] += __shfl_xor_sync(0xffffffffu, l_sum[nb][r], 16);
      }
    }
    if (consumers_any<kWarps * 32>(!ok || *guard.abort_flag != 0)) break;
#pragma unroll
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 8 * nb + 2 * t4 + r;
        if (row >= rows) continue;
        if (g == 0) {
          join_m[warp * kRows + row] = m_ref[nb][r];
          join_l[warp * kRows + row] = l_sum[nb][r];
        }
        float* dst = join_o + (warp * kRows + row) * D + 2 * g;
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
          *reinterpret_cast<float2*>(dst + 16 * c) = make_float2(o[nb][c][r], o[nb][c][2 + r]);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kWarps * 32) {
      const int row = idx / (D / 4), col = (idx % (D / 4)) * 4;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, join_m[w * kRows + row]);
      const float top = m == -INFINITY ? 0.f : m;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float d = join_m[w * kRows + row] - top, f = ex2(d);
        const float4 x = *reinterpret_cast<const float4*>(join_o + (w * kRows + row) * D + col);
        l += scale_sum(join_l[w * kRows + row], d);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
        acc.z = fmaf(x.z, f, acc.z);
        acc.w = fmaf(x.w, f, acc.w);
      }
      const int token = row / a.group, head = s.hkv * a.group + row - token * a.group;
      const int64_t out_row = s.seq.row0 + s.first + token;
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* dst = static_cast<T*>(a.o) + out_row * a.o_stride[0] + head * a.o_stride[1] + col;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv),
                                                    pack2<T>(acc.z * inv, acc.w * inv));
        if (col == 0)
          a.lse[out_row * a.heads + head] =
              l == 0.f ? -INFINITY : m * 0.69314718055994530942f + logf(l);
      } else {
        *reinterpret_cast<float4*>(a.part_o + ((static_cast<int64_t>(slot) * (D / 8) + col / 8) *
                                                   a.part_rows + row) * 8 + col % 8) = acc;
        if (col == 0)
          reinterpret_cast<float2*>(a.part_ml)[static_cast<int64_t>(slot) * a.part_rows + row] =
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
}

template <typename T, int D, int kBlocks>
int launch(const ExtendArgs& a, const QueryView& qv, const CUtensorMap& tmk, const CUtensorMap& tmv,
           int ctas, int dev, cudaStream_t stream) {
  using G = FewGeometry<D, kBlocks>;
  constexpr int kSmem = G::kTailOffset + static_cast<int>(sizeof(FewShared<G::kStages>)) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
  static thread_local int configured_device = -1;
  if (configured_device != dev) {
    if (int st = check_cuda(cudaFuncSetAttribute(extend_few_kernel<T, D, kBlocks>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSmem),
                            "cudaFuncSetAttribute(extend few)"))
      return st;
    configured_device = dev;
  }
  extend_few_kernel<T, D, kBlocks><<<ctas, G::kThreads, kSmem, stream>>>(a, qv, tmk, tmv);
  return check_cuda(cudaGetLastError(), "extend_few_kernel launch");
}

template <typename T>
int launch_t(const ExtendArgs& a, const QueryView& qv, const CUtensorMap& tmk,
             const CUtensorMap& tmv, int head_dim, int rows, int ctas, int dev,
             cudaStream_t stream) {
  if (head_dim == 128)
    return rows <= 8 ? launch<T, 128, 1>(a, qv, tmk, tmv, ctas, dev, stream)
                     : launch<T, 128, 2>(a, qv, tmk, tmv, ctas, dev, stream);
  return rows <= 8 ? launch<T, 64, 1>(a, qv, tmk, tmv, ctas, dev, stream)
                   : launch<T, 64, 2>(a, qv, tmk, tmv, ctas, dev, stream);
}

}  // namespace

int launch_extend_few(const ExtendArgs& args, const flb_kv_cache* c, const void* q,
                      int64_t q_row_stride, int64_t q_head_stride, int dtype, int ctas, int dev,
                      cudaStream_t stream) {
  ExtendArgs a = args;
  // Four keys' scales as one 16-byte load: contiguous along the keys and aligned at every fourth
  // key (a page, like a tile, starts at a multiple of 4 keys).
  auto wide = [](const float* base, const int64_t (&stride)[3]) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride[1] == 1 && stride[0] % 4 == 0 &&
           stride[2] % 4 == 0;
  };
  a.wide_scales = wide(a.cache.ks, a.cache.ks_stride) && wide(a.cache.vs, a.cache.vs_stride);
  const QueryView qv{q, {q_row_stride, q_head_stride}};
  CUtensorMap tmk, tmv;
  const int d = c->head_dim;
  View4 kv = kv_view4(c, false), vv = kv_view4(c, true);
  a.k_once = fold_expanded(&kv);
  a.v_once = fold_expanded(&vv);
  if (int st = encode_rows_map(&tmk, &a.kc, kv, a.box_rows, d, FLB_INT8, d)) return st;
  if (int st = encode_rows_map(&tmv, &a.vc, vv, a.box_rows, d, FLB_INT8, d)) return st;
  const int rows = a.tile_tokens * a.group;   // the most score rows of a sequence
  if (dtype == FLB_BF16)
    return launch_t<__nv_bfloat16>(a, qv, tmk, tmv, d, rows, ctas, dev, stream);
  return launch_t<__half>(a, qv, tmk, tmv, d, rows, ctas, dev, stream);
}

}  // namespace flb
