// Writing and reading a KV cache on sm_100a: flb_kv_append (new K/V rows into a contiguous or paged
// cache, quantised to 8 bits on the way when the cache is FLB_INT8) and flb_kv_gather (whole
// sequences back as 16- or 32-bit rows).
//
// The mathematics. A row x of D values (one token, one KV head) is stored as q = round(x r),
// r = min(127 (1 / a), 2^100), a = max|x|, with the scale s = max(a (1 / 127), 2^-100): |x - q s| is at
// most half a step s plus the fp32 roundings of 1 / a, r, x r and s. The bounds keep r and s finite and normal
// for rows of zeros and denormals (and 127 s finite at the largest values). Non-finite rows are stored as (0, NaN).
//
// Each byte moves once, so HBM should bound both directions (launch latency for single-token calls):
// at 6.5 TB/s an SM has 15 values of a 16-bit row per clock, which leaves about eight instructions per
// value and excludes the quarter-rate int <-> float conversions. Codes are rounded and read by
// adding 1.5 2^23 or 2^23 instead, whose last place is 1. A lane holds 16 bytes of each half of an
// outside row, so a row is D * size / 32 lanes and its maximum a shuffle reduction over them; with 16
// bytes per lane and row the addresses cost more than the values. Finding where
// a token lives takes three or four dependent loads (offsets, length, block table); one warp
// does it for the block's tokens while the others' first rows are on their way (append), and
// the rows then stream. Measured on B200 (H_kv 8, D 128, bf16 rows, int8 cache): append of 8 prompts of
// 900-3300 tokens 51 us, 4.9 TB/s; gather of 8 sequences of 5000-16384 keys 95 us, 5.9 TB/s; fp16
// without codes (H_kv 32, D 64, 110 MB) 21 us, 5.4 TB/s.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kv_cache.cuh"
#include "sm100.cuh"

namespace flb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTokens = 8;         // of one block (32: 5 % slower): a lane of its first warp finds
                                      // each one's place
constexpr int kBlocksAtLeast = 592;   // four per SM
constexpr float kStep = 1.f / 127.f;
constexpr float kMinScale = 0x1p-100f;
constexpr float kMaxInverse = 0x1p+100f;
constexpr float kMaxScale = 0x1.020406p+121f;   // the largest s with 127 s finite in fp32

struct RowsView {
  char* k;
  char* v;
  int64_t k_stride[2], v_stride[2];   // row, head (elements)
  const int32_t* seq_lens;
  Ragged ragged;
};

constexpr float kRoundBias = 12582912.f;   // 1.5 2^23: x + kRoundBias has round(x) in its low bits

// The 16-byte chunk of a row as floats (8 of a 16-bit type, 4 of fp32).
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& c, float (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// The largest magnitude of the chunk as the bits of a float, where infinities and NaN exceed every
// finite value.
template <typename T>
__device__ __forceinline__ uint32_t largest(const uint4& c) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  if constexpr (std::is_same<T, float>::value) {
    return max(max(w[0] & 0x7fffffffu, w[1] & 0x7fffffffu),
               max(w[2] & 0x7fffffffu, w[3] & 0x7fffffffu));
  } else {
    // NaN-propagating maxima of pairs.
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2,
                                         __nv_bfloat162>::type;
    T2 top = __habs2(*reinterpret_cast<const T2*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&w[i])));
    const float lo = static_cast<float>(top.x), hi = static_cast<float>(top.y);
    return max(__float_as_uint(lo) & 0x7fffffffu, __float_as_uint(hi) & 0x7fffffffu);
  }
}

// The codes round(x inv) of four values, in the bytes of a word.
__device__ __forceinline__ uint32_t encode4(const float* x, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), kRoundBias));
  return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// The values q s of the four codes of a word.
__device__ __forceinline__ void decode4(uint32_t codes, float scale, float (&x)[4]) {
  codes ^= 0x80808080u;   // 128 + q
  // Bytes over the bits of 2^23: 2^23 + 128 + q.
  const float f0 = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7440));
  const float f1 = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7441));
  const float f2 = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7442));
  const float f3 = __uint_as_float(__byte_perm(codes, 0x4b000000u, 0x7443));
  fadd2(x[0], x[1], f0, f1, -8388736.f, -8388736.f);
  fadd2(x[2], x[3], f2, f3, -8388736.f, -8388736.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] *= scale;
}

// A block moves the 2 H_kv rows (slots: the heads of K, then the heads of V) of `tokens` consecutive
// tokens. kAppend: outside rows into the cache, else the cache into outside rows.
template <typename T, int D, bool kQuant, bool kAppend>
__global__ void __launch_bounds__(kThreads) kv_move_kernel(const __grid_constant__ KvView c,
                                                           const __grid_constant__ RowsView r,
                                                           const __grid_constant__ FastDiv slots,
                                                           int tokens) {
  constexpr int kPer = 16 / sizeof(T);          // values of 16 bytes
  constexpr int kLanes = D / (2 * kPer);        // lanes per row: 16 bytes of each half
  constexpr int kRows = 32 / kLanes;            // rows per warp and step
  constexpr int kSteps = kQuant ? 2 : 4;        // steps whose loads are issued together
  // Where each token's rows are in the cache and in its scales (K, V, scales of K, of V); -1: nowhere.
  __shared__ int64_t place[kMaxTokens][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / kLanes, at = lane % kLanes;
  const int t0 = blockIdx.x * tokens;
  const int rows = min(tokens, r.ragged.rows - t0) * slots.d;

  struct Row {
    int token, h;   // within the block; head
    bool in, is_v;
  };
  auto row_at = [&](int step, int i) {
    const int x = ((step * kSteps + i) * kWarps + warp) * kRows + sub;
    Row row;
    row.in = x < rows;
    row.token = row.in ? slots.div(x) : 0;
    const int slot = x - row.token * slots.d;
    row.is_v = slot >= c.heads_kv;
    row.h = row.is_v ? slot - c.heads_kv : slot;
    return row;
  };
  struct Data {
    uint4 half[2];
    float scale;
  };
  auto outside = [&](const Row& x) {   // and D / 2 values on
    const int64_t t = t0 + x.token;
    return x.is_v ? reinterpret_cast<T*>(r.v) + t * r.v_stride[0] + x.h * r.v_stride[1] + at * kPer
                  : reinterpret_cast<T*>(r.k) + t * r.k_stride[0] + x.h * r.k_stride[1] + at * kPer;
  };
  // A row as it comes: from outside (append), else codes or values of the cache.
  auto load = [&](const Row& x) {
    Data d;
    d.half[0] = d.half[1] = make_uint4(0, 0, 0, 0);
    d.scale = 0.f;
    if constexpr (kAppend) {
      if (x.in) {
        const T* from = outside(x);
        d.half[0] = __ldg(reinterpret_cast<const uint4*>(from));
        d.half[1] = __ldg(reinterpret_cast<const uint4*>(from + D / 2));
      }
    } else {
      const int64_t base = place[x.token][x.is_v];
      if (x.in && base >= 0) {
        const int64_t off = base + x.h * (x.is_v ? c.v_stride[2] : c.k_stride[2]) + at * kPer;
        const void* from = x.is_v ? c.v : c.k;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (!kQuant) {
            d.half[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(from) + off +
                                                        j * (D / 2));
          } else {
            const int8_t* src = static_cast<const int8_t*>(from) + off + j * (D / 2);
            if constexpr (kPer == 8) {
              const uint2 w = *reinterpret_cast<const uint2*>(src);
              d.half[j].x = w.x;
              d.half[j].y = w.y;
            } else {
              d.half[j].x = *reinterpret_cast<const uint32_t*>(src);
            }
          }
        }
        if constexpr (kQuant)
          d.scale = (x.is_v ? c.vs : c.ks)[place[x.token][2 + x.is_v] +
                                           x.h * (x.is_v ? c.vs_stride[2] : c.ks_stride[2])];
      }
    }
    return d;
  };
  auto store = [&](const Row& x, const Data& d) {
    if constexpr (!kAppend) {
      T* to = outside(x);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint4 out = d.half[j];
        if constexpr (kQuant) {
          float y[4];
          decode4(d.half[j].x, d.scale, y);
          if constexpr (kPer == 8) {
            float z[4];
            decode4(d.half[j].y, d.scale, z);
            out = make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(z[0], z[1]),
                             pack2<T>(z[2], z[3]));
          } else {
            out = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                             __float_as_uint(y[3]));
          }
        }
        if (x.in) *reinterpret_cast<uint4*>(to + j * (D / 2)) = out;
      }
    } else {
      const int64_t base = place[x.token][x.is_v];
      const bool in = x.in && base >= 0;
      const int64_t off = base + x.h * (x.is_v ? c.v_stride[2] : c.k_stride[2]) + at * kPer;
      void* to = x.is_v ? c.v : c.k;
      if constexpr (!kQuant) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (in) *reinterpret_cast<uint4*>(static_cast<T*>(to) + off + j * (D / 2)) = d.half[j];
        }
      } else {
        uint32_t top = max(largest<T>(d.half[0]), largest<T>(d.half[1]));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
          top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float amax = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;
        const float inv = fminf(__fmul_rn(127.f, __frcp_rn(amax)), kMaxInverse);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float y[kPer];
          unpack16<T>(d.half[j], y);
          uint32_t q[kPer / 4];
#pragma unroll
          for (int e = 0; e < kPer / 4; ++e) q[e] = finite ? encode4(y + 4 * e, inv) : 0u;
          int8_t* dst = static_cast<int8_t*>(to) + off + j * (D / 2);
          if (in) {
            if constexpr (kPer == 8) {
              *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
            } else {
              *reinterpret_cast<uint32_t*>(dst) = q[0];
            }
          }
        }
        if (in && at == 0)
          (x.is_v ? c.vs : c.ks)[place[x.token][2 + x.is_v] +
                                 x.h * (x.is_v ? c.vs_stride[2] : c.ks_stride[2])] =
              finite ? fminf(fmaxf(__fmul_rn(amax, kStep), kMinScale), kMaxScale)
                     : __uint_as_float(0x7fffffffu);
      }
    }
  };

  constexpr int kAtOnce = kSteps * kWarps * kRows;   // rows per round of the loop below
  Row x[kSteps];
  Data d[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    x[i] = row_at(0, i);
    if (kAppend) d[i] = load(x[i]);   // does not depend on the places
  }
  if (warp == 0) {   // lanes past the block's tokens look up rows of the next one
    int b, at_row, count;
    int64_t outer = 0, row = 0;
    const bool owned = find_sequences(r.ragged, t0, lane, b, at_row, count) && lane < tokens;
    int pos = -1;
    if (owned) {
      const int len = __ldg(r.seq_lens + b);
      pos = kAppend ? len - count + at_row : at_row < len ? at_row : -1;
    }
    const bool here = owned && c.locate(b, pos, outer, row);
    if (lane < kMaxTokens) {
      place[lane][0] = here ? outer * c.k_stride[0] + row * c.k_stride[1] : -1;
      place[lane][1] = here ? outer * c.v_stride[0] + row * c.v_stride[1] : -1;
      place[lane][2] = outer * c.ks_stride[0] + row * c.ks_stride[1];
      place[lane][3] = outer * c.vs_stride[0] + row * c.vs_stride[1];
    }
  }
  __syncthreads();
  for (int step = 0; step * kAtOnce < rows; ++step) {
    if (step > 0 || !kAppend) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        x[i] = row_at(step, i);
        d[i] = load(x[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) store(x[i], d[i]);
  }
}

template <typename T, int D, bool kQuant>
int launch(const KvView& c, const RowsView& r, bool append, cudaStream_t stream) {
  // Tokens per block: as many as leave kBlocksAtLeast blocks, so that few tokens spread over the GPU
  // and many share the look-up of their places.
  int tokens = 1;
  while (tokens < kMaxTokens && r.ragged.rows / (2 * tokens) >= kBlocksAtLeast) tokens *= 2;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(r.ragged.rows) + tokens - 1) /
                                              tokens);
  const FastDiv slots = FastDiv::of(2 * c.heads_kv);
  if (append)
    kv_move_kernel<T, D, kQuant, true><<<grid, kThreads, 0, stream>>>(c, r, slots, tokens);
  else
    kv_move_kernel<T, D, kQuant, false><<<grid, kThreads, 0, stream>>>(c, r, slots, tokens);
  return check_cuda(cudaGetLastError(), append ? "kv append launch" : "kv gather launch");
}

template <typename T>
int launch_t(const flb_kv_cache* c, const KvView& cv, const RowsView& rv, bool append,
             cudaStream_t stream) {
  const bool quant = c->dtype == FLB_INT8;
  if (c->head_dim == 128)
    return quant ? launch<T, 128, true>(cv, rv, append, stream)
                 : launch<T, 128, false>(cv, rv, append, stream);
  return quant ? launch<T, 64, true>(cv, rv, append, stream)
               : launch<T, 64, false>(cv, rv, append, stream);
}

int run(const flb_kv_cache* c, const flb_kv_rows* r, bool append, cudaStream_t stream) {
  clear_error();
  if (int st = validate_kv_cache(c)) return st;
  if (r == nullptr) return fail(FLB_ERR_INVALID_ARGUMENT, "rows is NULL");
  if (!r->k || !r->v || !r->seq_lens)
    return fail(FLB_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (r->rows <= 0 || (r->cu_seqlens == nullptr && r->rows_per_seq <= 0))
    return fail(FLB_ERR_INVALID_ARGUMENT, "empty input: %d rows, %d per sequence", r->rows,
                r->rows_per_seq);
  if (r->dtype != FLB_BF16 && r->dtype != FLB_FP16 && r->dtype != FLB_FP32)
    return fail(FLB_ERR_UNSUPPORTED, "rows are bf16, fp16 or fp32 (dtype code %d)", r->dtype);
  if (c->dtype != FLB_INT8 && c->dtype != r->dtype)
    return fail(FLB_ERR_UNSUPPORTED, "rows (dtype code %d) and cache (%d) differ", r->dtype,
                c->dtype);
  const int esize = r->dtype == FLB_FP32 ? 4 : 2;
  const View4 kv{r->k, {1, r->rows, c->heads_kv, c->head_dim},
                 {0, r->k_row_stride, r->k_head_stride, 1}, esize};
  const View4 vv{r->v, {1, r->rows, c->heads_kv, c->head_dim},
                 {0, r->v_row_stride, r->v_head_stride, 1}, esize};
  if (!rows_16b_aligned(kv))
    return fail(FLB_ERR_MISALIGNED, "k must have 16-byte aligned rows (data pointer and strides)");
  if (!rows_16b_aligned(vv))
    return fail(FLB_ERR_MISALIGNED, "v must have 16-byte aligned rows (data pointer and strides)");
  if (int st = current_device_info(nullptr, nullptr, nullptr, nullptr)) return st;
  RowsView rv{};
  rv.k = static_cast<char*>(r->k);
  rv.v = static_cast<char*>(r->v);
  rv.k_stride[0] = r->k_row_stride;
  rv.k_stride[1] = r->k_head_stride;
  rv.v_stride[0] = r->v_row_stride;
  rv.v_stride[1] = r->v_head_stride;
  rv.seq_lens = r->seq_lens;
  rv.ragged = Ragged{r->cu_seqlens, r->rows, r->rows_per_seq, c->batch};
  const KvView cv = kv_view(c);
  if (r->dtype == FLB_BF16) return launch_t<__nv_bfloat16>(c, cv, rv, append, stream);
  if (r->dtype == FLB_FP16) return launch_t<__half>(c, cv, rv, append, stream);
  return launch_t<float>(c, cv, rv, append, stream);
}

}  // namespace

int validate_kv_cache(const flb_kv_cache* c) {
  if (c == nullptr) return fail(FLB_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (!c->k_cache || !c->v_cache)
    return fail(FLB_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (c->batch <= 0 || c->heads_kv <= 0 || c->max_seqlen <= 0)
    return fail(FLB_ERR_INVALID_ARGUMENT, "empty cache: batch %d heads_kv %d S_max %d", c->batch,
                c->heads_kv, c->max_seqlen);
  if (c->max_seqlen > kMaxSeqlen)
    return fail(FLB_ERR_UNSUPPORTED, "S_max %d is more than %d", c->max_seqlen, kMaxSeqlen);
  if (c->dtype != FLB_BF16 && c->dtype != FLB_FP16 && c->dtype != FLB_FP32 &&
      c->dtype != FLB_INT8)
    return fail(FLB_ERR_UNSUPPORTED, "a cache is bf16, fp16, fp32 or int8 (dtype code %d)",
                c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(FLB_ERR_UNSUPPORTED, "unsupported head_dim %d (64 or 128)", c->head_dim);
  if ((c->dtype == FLB_INT8) != (c->k_scale != nullptr) ||
      (c->dtype == FLB_INT8) != (c->v_scale != nullptr))
    return fail(FLB_ERR_INVALID_ARGUMENT,
                "an int8 cache needs k_scale and v_scale, any other cache takes neither");
  if (c->block_tables != nullptr) {
    if (c->page_size <= 0 || c->num_blocks <= 0)
      return fail(FLB_ERR_INVALID_ARGUMENT,
                  "paged cache: page_size %d and num_blocks %d must be positive", c->page_size,
                  c->num_blocks);
    if (c->max_seqlen % c->page_size != 0)
      return fail(FLB_ERR_INVALID_ARGUMENT,
                  "paged cache: max_seqlen %d must be max_blocks * page_size (page_size %d)",
                  c->max_seqlen, c->page_size);
    if (c->batch > 1 && c->block_table_stride < c->max_seqlen / c->page_size)
      return fail(FLB_ERR_INVALID_ARGUMENT, "paged cache: block_table_stride %lld < max_blocks %d",
                  static_cast<long long>(c->block_table_stride), c->max_seqlen / c->page_size);
  }
  if (!rows_16b_aligned(kv_view4(c, false)))
    return fail(FLB_ERR_MISALIGNED,
                "k_cache must have 16-byte aligned rows (data pointer and strides)");
  if (!rows_16b_aligned(kv_view4(c, true)))
    return fail(FLB_ERR_MISALIGNED,
                "v_cache must have 16-byte aligned rows (data pointer and strides)");
  return FLB_OK;
}

View4 kv_view4(const flb_kv_cache* c, bool v) {
  const bool paged = c->block_tables != nullptr;
  const int64_t outer = paged ? c->num_blocks : c->batch;
  const int64_t rows = paged ? c->page_size : c->max_seqlen;
  const int esize = c->dtype == FLB_INT8 ? 1 : c->dtype == FLB_FP32 ? 4 : 2;
  if (v)
    return View4{c->v_cache, {outer, rows, c->heads_kv, c->head_dim},
                 {c->v_batch_stride, c->v_seq_stride, c->v_head_stride, 1}, esize};
  return View4{c->k_cache, {outer, rows, c->heads_kv, c->head_dim},
               {c->k_batch_stride, c->k_seq_stride, c->k_head_stride, 1}, esize};
}

KvView kv_view(const flb_kv_cache* c) {
  KvView v{};
  v.k = c->k_cache;
  v.v = c->v_cache;
  v.ks = c->k_scale;
  v.vs = c->v_scale;
  const int64_t ks[3] = {c->k_batch_stride, c->k_seq_stride, c->k_head_stride};
  const int64_t vs[3] = {c->v_batch_stride, c->v_seq_stride, c->v_head_stride};
  const int64_t kss[3] = {c->ks_batch_stride, c->ks_seq_stride, c->ks_head_stride};
  const int64_t vss[3] = {c->vs_batch_stride, c->vs_seq_stride, c->vs_head_stride};
  for (int i = 0; i < 3; ++i) {
    v.k_stride[i] = ks[i];
    v.v_stride[i] = vs[i];
    v.ks_stride[i] = kss[i];
    v.vs_stride[i] = vss[i];
  }
  v.block_tables = c->block_tables;
  v.bt_stride = c->block_table_stride;
  const bool paged = c->block_tables != nullptr;
  v.page = FastDiv::of(paged ? c->page_size : 1);
  v.max_blocks = paged ? c->max_seqlen / c->page_size : 0;
  v.num_blocks = c->num_blocks;
  v.max_seqlen = c->max_seqlen;
  v.heads_kv = c->heads_kv;
  v.batch = c->batch;
  return v;
}

}  // namespace flb

extern "C" int flb_kv_append(const flb_kv_cache* cache, const flb_kv_rows* rows,
                             flb_stream_t stream) {
  return flb::run(cache, rows, true, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int flb_kv_gather(const flb_kv_cache* cache, const flb_kv_rows* rows,
                             flb_stream_t stream) {
  return flb::run(cache, rows, false, reinterpret_cast<cudaStream_t>(stream));
}
