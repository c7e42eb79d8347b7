// Attention of a few new rows per sequence over an int8 KV cache: single-token decode, and chunks
// whose (tokens x query heads of one KV head) are at most 16 score rows. Same operator, work split
// and partials as extend.cu; HBM bound (2 H_kv (D + 4) bytes per key), so the codes go from shared
// memory straight into the registers of 16 x 8 x 16 warp MMAs instead of through 16-bit tiles (the
// tcgen05 form of extend.cu took 297 us for 8 sequences of 24K keys, H_kv 8, D 128).
//
//  * One CTA per SM: one warp streams [128 keys x D] tiles of K and V codes by TMA, another turns the
//    keys' scales into what the scores need (below) beside them in the ring stage, and eight
//    consumer warps take 16 keys of every tile, each with its own online softmax; their results
//    are joined in a fixed order at the end of a segment. Block tables are read 32 entries at a
//    time. (One producer warp for copies and scales, with a table load per key, bounded 16-row
//    pages: 5000 clocks per tile where the consumers took 2400.)
//  * Q is the A operand (rows = tokens x heads), in fp16: bf16 queries are scaled to [1, 2) of
//    their row's maximum by a power of two, which is exact down to 2^-17 of the maximum and off by at
//    most 2^-25 of it below. The order of a dot product is free, so thread t of a quad takes D / 4
//    consecutive values of its key's row (16-byte shared loads) and the same ones of Q.
//  * V goes through transposed 8 x 8 matrix loads of byte pairs: a register then holds columns d and
//    d + 1 of two keys, one fragment for the even and one for the odd columns.
//  * The scales act as in extend.cu: z = s mult + log2 sv, w = 2^(z - M) in fp16, the row sum takes
//    w / sv.
#include <algorithm>

#include "extend_work.cuh"

namespace flb {
namespace {

constexpr int kWarps = 8;             // consumers: 16 keys of a tile each
constexpr int kCopyWarp = kWarps;      // TMA of the codes
constexpr int kScaleWarp = kWarps + 1;
constexpr int kFewThreads = (kWarps + 2) * 32;
static_assert(kWarps * 16 == kBN, "the consumers cover a tile");

template <int D>
struct FewGeometry {
  static constexpr int kTileBytes = kBN * D;          // K or V codes
  static constexpr int kStages = D == 128 ? 4 : 8;    // 128 KB of codes
  static constexpr int kScaleOffset = kStages * 2 * kTileBytes;
  static constexpr int kScaleBytes = 3 * kBN * 4;     // sk, log2 sv and 1 / sv of one stage
  static constexpr int kJoinOffset = kScaleOffset + kStages * kScaleBytes;
  static constexpr int kJoinBytes = kWarps * kFewTile * (D + 2) * 4;
  static constexpr int kTailOffset = kJoinOffset + kJoinBytes;
  static_assert((kMaxBatch + 1) * 8 <= kScaleOffset, "prefix sums fit in the ring");
};

template <int kStages>
struct FewShared {
  uint64_t full[kStages];
  uint64_t empty[kStages];
  int abort_flag;
  Share share;
};

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// True on all consumer threads when pred holds on any of them.
__device__ __forceinline__ bool consumers_any(bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(pred)), "n"(kWarps * 32)
      : "memory");
  return r != 0;
}

struct QueryView {
  const void* q;
  int64_t stride[2];   // row, head
};

template <typename T, int D>
__global__ void __launch_bounds__(kFewThreads, 1)
    extend_few_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ QueryView qv,
                      const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using G = FewGeometry<D>;
  constexpr int kStages = G::kStages;
  constexpr int kSteps = D / 16;    // MMA steps over head_dim
  constexpr int kCols = D / 8;      // 8-column blocks of O
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  auto* sh = reinterpret_cast<FewShared<kStages>*>(smem + G::kTailOffset);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    sh->abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh->full[i], 33);   // the TMA bytes and each lane's scales
      mbar_init(&sh->empty[i], kWarps);
    }
    fence_barrier_init();
  }
  if (warp == kCopyWarp && lane == 0) {
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  find_share(a, &sh->share, reinterpret_cast<int64_t*>(smem));
  fence_proxy_async_shared();   // the ring was written here; TMA writes it next
  __syncthreads();
  const WaitGuard guard{reinterpret_cast<volatile int*>(&sh->abort_flag), a.status};
  Walk walk;
  Segment s;
  walk.start(a, sh->share);

  if (warp == kCopyWarp) {
    // ------------------------------- copies -------------------------------
    // Lane i issues copy i of a tile: a part of box_rows rows, of K or of V.
    const int parts = kBN / a.box_rows;
    const bool issues = lane < 2 * parts;
    const bool is_v = lane >= parts;
    const int offset = (is_v ? lane - parts : lane) % parts * a.box_rows;   // of the part's keys
    const bool paged = a.cache.block_tables != nullptr;
    const CUtensorMap* map = is_v ? &tmv : &tmk;
    const TmaCoords& c = is_v ? a.vc : a.kc;
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
          blk = window.at(page);
          row = key - page * a.cache.page.d;
        }
        const int st = issued % kStages;
        ok = issued < kStages || mbar_wait(&sh->empty[st], ((issued / kStages) - 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&sh->full[st], 2 * G::kTileBytes);
        __syncwarp();
        if (issues)
          tma_load_4d(smem + (2 * st + (is_v ? 1 : 0)) * G::kTileBytes + offset * D, map,
                      &sh->full[st], 0, tma_c(c, 1, row, s.hkv, blk), tma_c(c, 2, row, s.hkv, blk),
                      tma_c(c, 3, row, s.hkv, blk));
        ++issued;
      }
    }
    // Wait for the copies still landing before the CTA may exit.
    for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
      if (!mbar_wait(&sh->full[i % kStages], (i / kStages) & 1, guard)) break;
    }
    return;
  }
  if (warp == kScaleWarp) {
    // ------------------------------- scales -------------------------------
    // Lane i turns the scales of keys 4 i .. 4 i + 3 of a tile, read one tile ahead, into sk,
    // log2 sv and 1 / sv. They lie in one page. With a.wide_scales they are 16 contiguous bytes.
    const bool paged = a.cache.block_tables != nullptr;
    const int64_t ks_row = a.cache.ks_stride[1], vs_row = a.cache.vs_stride[1];
    BlockWindow window;
    int issued = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      if (paged) window.start(a.cache, s.b, a.cache.page.div(s.t0 * kBN), lane);
      // Keys past the length are not read: they stay hidden, whatever their scales.
      auto fetch = [&](int tile, float (&sk)[4], float (&sv)[4]) {
        const int key = tile * kBN + 4 * lane;
        int64_t outer = s.b, row = key;
        if (paged) {
          const int page = a.cache.page.div(key);
          window.advance(a.cache, __shfl_sync(0xffffffffu, page, 0), lane);
          outer = window.at(page);
          row = key - page * a.cache.page.d;
        }
        const int keys = outer >= 0 ? s.seq.len - key : 0;
        const float* k = a.cache.ks + outer * a.cache.ks_stride[0] + row * ks_row +
                         s.hkv * a.cache.ks_stride[2];
        const float* v = a.cache.vs + outer * a.cache.vs_stride[0] + row * vs_row +
                         s.hkv * a.cache.vs_stride[2];
        if (a.wide_scales && keys >= 4) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(k));
          const float4 y = __ldg(reinterpret_cast<const float4*>(v));
          sk[0] = x.x, sk[1] = x.y, sk[2] = x.z, sk[3] = x.w;
          sv[0] = y.x, sv[1] = y.y, sv[2] = y.z, sv[3] = y.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sk[i] = i < keys ? __ldg(k + i * ks_row) : 0.f;
            sv[i] = i < keys ? __ldg(v + i * vs_row) : kMinScale;
          }
        }
      };
      float sk[4], sv[4];
      if (s.t0 < s.t1) fetch(s.t0, sk, sv);
      for (int tile = s.t0; tile < s.t1; ++tile) {
        float sk_next[4] = {0.f, 0.f, 0.f, 0.f}, sv_next[4] = {0.f, 0.f, 0.f, 0.f};
        if (tile + 1 < s.t1) fetch(tile + 1, sk_next, sv_next);
        const int st = issued % kStages;
        ok = issued < kStages || mbar_wait(&sh->empty[st], ((issued / kStages) - 1) & 1, guard);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float add[4], inv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = sv[i] < kMinScale ? kMinScale : sv[i];
          add[i] = lg2(v);
          // A scale that is not finite reaches the rows that see its key through z only.
          inv[i] = v <= 0x1p+127f ? rcp(v) : 0.f;
        }
        float4* dst = reinterpret_cast<float4*>(smem + G::kScaleOffset + st * G::kScaleBytes) + lane;
        dst[0] = make_float4(sk[0], sk[1], sk[2], sk[3]);
        dst[kBN / 4] = make_float4(add[0], add[1], add[2], add[3]);
        dst[2 * (kBN / 4)] = make_float4(inv[0], inv[1], inv[2], inv[3]);
        mbar_arrive(&sh->full[st]);
        ++issued;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sk[i] = sk_next[i];
          sv[i] = sv_next[i];
        }
      }
    }
    zero_other_rows<T, D>(a, blockIdx.x, gridDim.x, lane);
    return;
  }

  // ------------------------------- consumers -------------------------------
  const int g = lane >> 2;    // fragment row group
  const int t4 = lane & 3;    // thread in quad
  float* join_m = reinterpret_cast<float*>(smem + G::kJoinOffset);   // [warps][16]
  float* join_l = join_m + kWarps * kFewTile;
  float* join_o = join_l + kWarps * kFewTile;                        // [warps][16][D]
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t v_row = static_cast<uint32_t>(warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7));
  const uint32_t v_chunk = static_cast<uint32_t>(lane >> 4);
  int done = 0;               // tiles consumed
  int segments = 0;
  int4 meta0 = make_int4(0, 0, 0, 0), meta1 = make_int4(0, 0, 0, 0);
  bool ok = true;
  while (walk.next(a, s)) {
    const bool first_segment = segments++ == 0;
    const int rows = s.tokens * a.group;
    // Q fragments: rows g and g + 8, values [t4 D / 4, (t4 + 1) D / 4).
    uint32_t qa[kSteps][4];
    float row_scale[2] = {a.scale_log2, a.scale_log2};
    int limit[2];             // keys that the row sees
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      const int token = row / a.group, head = s.hkv * a.group + row - token * a.group;
      limit[r] = a.causal ? min(s.seq.len, s.seq.len - s.seq.n + s.first + token + 1) : s.seq.len;
      const uint2* src = reinterpret_cast<const uint2*>(
          static_cast<const T*>(qv.q) + (s.seq.row0 + s.first + token) * qv.stride[0] +
          head * qv.stride[1] + t4 * (D / 4));
      uint2 x[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) x[k] = row < rows ? __ldg(src + k) : make_uint2(0, 0);
      if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qa[k][r] = x[k].x;
          qa[k][2 + r] = x[k].y;
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
        row_scale[r] *= __uint_as_float(static_cast<uint32_t>(e) << 23);
        auto half_pair = [&](uint32_t v) {
          return pack2<__half>(__uint_as_float(v << 16) * down,
                               __uint_as_float(v & 0xffff0000u) * down);
        };
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          qa[k][r] = half_pair(x[k].x);
          qa[k][2 + r] = half_pair(x[k].y);
        }
      }
    }
    float o[kCols][4];        // block 2 c + p: columns 16 c + 2 n + p of chunk c, n = 0..7
#pragma unroll
    for (int i = 0; i < kCols; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_ref[2] = {-INFINITY, -INFINITY};   // log2-domain reference points
    float l_sum[2] = {0.f, 0.f};               // this thread's share of the row sums

    for (int tile = s.t0; ok && tile < s.t1; ++tile) {
      const int st = done % kStages;
      ok = mbar_wait(&sh->full[st], (done / kStages) & 1, guard);
      if (!ok) break;
      ++done;
      const uint8_t* kt = smem + 2 * st * G::kTileBytes;
      const uint32_t vt = smem_base + (2 * st + 1) * G::kTileBytes;
      const float* scales = reinterpret_cast<const float*>(smem + G::kScaleOffset +
                                                           st * G::kScaleBytes);
      const int key0 = tile * kBN + warp * 16;   // this warp's first key

      // Two accumulators per 8 keys: a chain of D / 16 dependent MMAs is half as long.
      float z[2][4], y[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const uint32_t row = warp * 16 + nt * 8 + g;
        uint4 x[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
          x[i] = *reinterpret_cast<const uint4*>(kt + code_offset<D>(row, t4 * (D / 64) + i));
#pragma unroll
        for (int e = 0; e < 4; ++e) z[nt][e] = y[nt][e] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          const uint32_t word[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t lo, hi;
            codes_to_16bit<__half>(word[w], lo, hi);
            mma_16816<__half>((w & 1) ? y[nt] : z[nt], qa[4 * i + w], lo, hi);
          }
        }
      }
      // Keys nt * 8 + 2 t4 + {0, 1} of this warp.
      float2 inv[2];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const float* at = scales + warp * 16 + nt * 8 + 2 * t4;
        const float2 sk = *reinterpret_cast<const float2*>(at);
        const float2 add = *reinterpret_cast<const float2*>(at + kBN);
        inv[nt] = *reinterpret_cast<const float2*>(at + 2 * kBN);
        const int key = key0 + nt * 8 + 2 * t4;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float z0 = fmaf((z[nt][2 * r] + y[nt][2 * r]) * row_scale[r], sk.x, add.x);
          const float z1 = fmaf((z[nt][2 * r + 1] + y[nt][2 * r + 1]) * row_scale[r], sk.y, add.y);
          z[nt][2 * r] = key < limit[r] ? z0 : -INFINITY;
          z[nt][2 * r + 1] = key + 1 < limit[r] ? z1 : -INFINITY;
        }
      }
      float factor[2], ref[2];
      bool rescale = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = fmaxf(fmaxf(z[0][2 * r], z[0][2 * r + 1]), fmaxf(z[1][2 * r], z[1][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // The reference point moves only when the maximum passes it by more than 2^8.
        float m_new = m_ref[r];
        if (m_new == -INFINITY || mx > m_new + kRescaleThreshold) m_new = fmaxf(m_new, mx);
        factor[r] = 1.f;
        if (m_new != m_ref[r]) {
          factor[r] = ex2(m_ref[r] - m_new);   // 0 for the first keys
          rescale = true;
        }
        m_ref[r] = m_new;
        ref[r] = m_new == -INFINITY ? 0.f : m_new;
      }
      if (__any_sync(0xffffffffu, rescale)) {
        l_sum[0] *= factor[0];
        l_sum[1] *= factor[1];
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
          o[i][0] *= factor[0];
          o[i][1] *= factor[0];
          o[i][2] *= factor[1];
          o[i][3] *= factor[1];
        }
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) z[nt][e] = ex2(z[nt][e] - ref[e >> 1]);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          l_sum[r] = fmaf(z[nt][2 * r], inv[nt].x, fmaf(z[nt][2 * r + 1], inv[nt].y, l_sum[r]));
      }
      const uint32_t pa[4] = {pack2<__half>(z[0][0], z[0][1]), pack2<__half>(z[0][2], z[0][3]),
                              pack2<__half>(z[1][0], z[1][1]), pack2<__half>(z[1][2], z[1][3])};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[4];   // keys 0-7 and 8-15 of chunk 2 c, then of chunk 2 c + 1
        ldsm_x4_trans(vt + code_offset<D>(v_row, 2 * c + v_chunk), v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t even0, odd0, even1, odd1;
          code_columns(v[2 * half], even0, odd0);
          code_columns(v[2 * half + 1], even1, odd1);
          mma_16816<__half>(o[2 * (2 * c + half)], pa, even0, even1);
          mma_16816<__half>(o[2 * (2 * c + half) + 1], pa, odd0, odd1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->empty[st]);
    }

    // Join the warps. Every consumer is past the previous segment's reads after the first barrier.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 1);
      l_sum[r] += __shfl_xor_sync(0xffffffffu, l_sum[r], 2);
    }
    if (consumers_any(!ok || *guard.abort_flag != 0)) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r;
      if (row >= rows) continue;
      if (t4 == 0) {
        join_m[warp * kFewTile + row] = m_ref[r];
        join_l[warp * kFewTile + row] = l_sum[r];
      }
      float* dst = join_o + (warp * kFewTile + row) * D;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        // Columns 16 c + 4 t4 + {0, 1, 2, 3}: even and odd blocks interleaved.
        *reinterpret_cast<float4*>(dst + 16 * c + 4 * t4) =
            make_float4(o[2 * c][2 * r], o[2 * c + 1][2 * r], o[2 * c][2 * r + 1],
                        o[2 * c + 1][2 * r + 1]);
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
    const bool whole = s.t0 == 0 && s.t1 == s.tiles;
    const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kWarps * 32) {
      const int row = idx / (D / 4), col = (idx % (D / 4)) * 4;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, join_m[w * kFewTile + row]);
      const float top = m == -INFINITY ? 0.f : m;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(join_m[w * kFewTile + row] - top);
        const float4 x = *reinterpret_cast<const float4*>(join_o + (w * kFewTile + row) * D + col);
        l = fmaf(join_l[w * kFewTile + row], f, l);
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

template <typename T, int D>
int launch(const ExtendArgs& a, const QueryView& qv, const CUtensorMap& tmk, const CUtensorMap& tmv,
           int ctas, int dev, cudaStream_t stream) {
  using G = FewGeometry<D>;
  constexpr int kSmem = G::kTailOffset + static_cast<int>(sizeof(FewShared<G::kStages>)) + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
  static thread_local int configured_device = -1;
  if (configured_device != dev) {
    if (int st = check_cuda(cudaFuncSetAttribute(extend_few_kernel<T, D>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 kSmem),
                            "cudaFuncSetAttribute(extend few)"))
      return st;
    configured_device = dev;
  }
  extend_few_kernel<T, D><<<ctas, kFewThreads, kSmem, stream>>>(a, qv, tmk, tmv);
  return check_cuda(cudaGetLastError(), "extend_few_kernel launch");
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
  if (int st = encode_rows_map(&tmk, &a.kc, kv_view4(c, false), a.box_rows, d, FLB_INT8, d))
    return st;
  if (int st = encode_rows_map(&tmv, &a.vc, kv_view4(c, true), a.box_rows, d, FLB_INT8, d))
    return st;
  if (dtype == FLB_BF16)
    return d == 128 ? launch<__nv_bfloat16, 128>(a, qv, tmk, tmv, ctas, dev, stream)
                    : launch<__nv_bfloat16, 64>(a, qv, tmk, tmv, ctas, dev, stream);
  return d == 128 ? launch<__half, 128>(a, qv, tmk, tmv, ctas, dev, stream)
                  : launch<__half, 64>(a, qv, tmk, tmv, ctas, dev, stream);
}

}  // namespace flb
