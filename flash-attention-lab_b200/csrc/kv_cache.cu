// Writing and reading a KV cache on sm_100a: flb_kv_append (new K/V rows into a contiguous or paged
// cache, quantised to 8 bits on the way when the cache is FLB_INT8) and flb_kv_gather (whole
// sequences back as 16- or 32-bit rows).
//
// The mathematics. A row x of D values (one token, one KV head) is stored as q = round(x r),
// r = min(127 / a, 2^100), a = max|x|, with the scale s = max(a / 127, 2^-100): |x - q s| is at most
// half a step s plus the fp32 roundings of r, x r and s. The bounds keep r and s finite and normal
// for rows of zeros and denormals (and 127 s finite at the largest values). Non-finite rows are stored as (0, NaN).
//
// Both kernels move each byte once and do a handful of operations per value, so HBM bounds them
// (launch latency for single-token calls). A warp handles one token and several of its 2 H_kv
// (K or V, head) rows; 16 bytes of a row per lane, so a row is D * size / 16 lanes and its
// maximum a shuffle reduction over them. The rows' loads are issued before the token's sequence
// is looked up (append), which takes two or three dependent loads (offsets, length, block table).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "kv_cache.cuh"
#include "sm100.cuh"

namespace flb {
namespace {

constexpr int kThreads = 128;
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

// The 16-byte chunk of a row as floats (8 of a 16-bit type, 4 of fp32) and back.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& c, float (&x)[16 / sizeof(T)]) {
  const T* e = reinterpret_cast<const T*>(&c);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) x[i] = static_cast<float>(e[i]);
}

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
  return (a & 0xff) | ((b & 0xff) << 8) | ((c & 0xff) << 16) | (static_cast<uint32_t>(d) << 24);
}

// Slot s of a token's 2 H_kv rows: the heads of K, then the heads of V.
template <typename T, int D, bool kQuant, int kIter>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ KvView c,
                                                             const __grid_constant__ RowsView r) {
  constexpr int kPer = 16 / sizeof(T);          // values per lane
  constexpr int kLanes = D / kPer;              // lanes per row
  constexpr int kRows = 32 / kLanes;            // rows per warp and iteration
  const int lane = threadIdx.x & 31;
  const int sub = lane / kLanes, at = lane % kLanes;
  const int slots = 2 * c.heads_kv;
  const int warps_per_token = (slots + kRows * kIter - 1) / (kRows * kIter);
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t token = w / warps_per_token;
  if (token >= r.ragged.rows) return;
  const int t = static_cast<int>(token);
  const int slot0 = static_cast<int>(w - token * warps_per_token) * (kRows * kIter);

  uint4 in[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int slot = slot0 + i * kRows + sub;
    const bool is_v = slot >= c.heads_kv;
    const int h = is_v ? slot - c.heads_kv : slot;
    in[i] = make_uint4(0, 0, 0, 0);
    if (slot < slots) {
      const int64_t off = is_v ? t * r.v_stride[0] + h * r.v_stride[1]
                               : t * r.k_stride[0] + h * r.k_stride[1];
      in[i] = __ldg(reinterpret_cast<const uint4*>(is_v ? r.v : r.k) +
                    (off + at * kPer) / kPer);
    }
  }
  int b, first, count;
  if (!find_sequence(r.ragged, t, lane, b, first, count)) return;
  int64_t outer, row;
  if (!c.locate(b, __ldg(r.seq_lens + b) - count + (t - first), outer, row)) return;

#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int slot = slot0 + i * kRows + sub;
    const bool is_v = slot >= c.heads_kv;
    const int h = is_v ? slot - c.heads_kv : slot;
    const int64_t* cs = is_v ? c.v_stride : c.k_stride;
    const int64_t off = outer * cs[0] + row * cs[1] + h * cs[2] + at * kPer;
    if constexpr (!kQuant) {
      if (slot < slots) *reinterpret_cast<uint4*>(static_cast<T*>(is_v ? c.v : c.k) + off) = in[i];
    } else {
      float x[kPer];
      unpack16<T>(in[i], x);
      // The largest magnitude as bits, where infinities and NaN exceed every finite value.
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float amax = __uint_as_float(top);
      const bool finite = top < 0x7f800000u;
      const float inv = fminf(__fdiv_rn(127.f, amax), kMaxInverse);
      int q[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        q[e] = finite ? max(-127, min(127, __float2int_rn(__fmul_rn(x[e], inv)))) : 0;
      if (slot < slots) {
        int8_t* dst = static_cast<int8_t*>(is_v ? c.v : c.k) + off;
        if constexpr (kPer == 8) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_codes(q[0], q[1], q[2], q[3]),
                                                      pack_codes(q[4], q[5], q[6], q[7]));
        } else {
          *reinterpret_cast<uint32_t*>(dst) = pack_codes(q[0], q[1], q[2], q[3]);
        }
        if (at == 0) {
          const int64_t* ss = is_v ? c.vs_stride : c.ks_stride;
          (is_v ? c.vs : c.ks)[outer * ss[0] + row * ss[1] + h * ss[2]] =
              finite ? fminf(fmaxf(__fdiv_rn(amax, 127.f), kMinScale), kMaxScale)
                     : __uint_as_float(0x7fffffffu);
        }
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ T from_float(float x) {
  return static_cast<T>(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
  return __float2half_rn(x);
}

template <typename T, int D, bool kQuant, int kIter>
__global__ void __launch_bounds__(kThreads) kv_gather_kernel(const __grid_constant__ KvView c,
                                                             const __grid_constant__ RowsView r) {
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kLanes = D / kPer;
  constexpr int kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const int sub = lane / kLanes, at = lane % kLanes;
  const int slots = 2 * c.heads_kv;
  const int warps_per_token = (slots + kRows * kIter - 1) / (kRows * kIter);
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t token = w / warps_per_token;
  if (token >= r.ragged.rows) return;
  const int t = static_cast<int>(token);
  const int slot0 = static_cast<int>(w - token * warps_per_token) * (kRows * kIter);

  int b = 0, first = 0, count = 0;
  int64_t outer = 0, row = 0;
  const bool found = find_sequence(r.ragged, t, lane, b, first, count) &&
                     t - first < __ldg(r.seq_lens + b) && c.locate(b, t - first, outer, row);
  uint4 raw[kIter];
  float scale[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int slot = slot0 + i * kRows + sub;
    const bool is_v = slot >= c.heads_kv;
    const int h = is_v ? slot - c.heads_kv : slot;
    raw[i] = make_uint4(0, 0, 0, 0);
    scale[i] = 0.f;
    if (found && slot < slots) {
      const int64_t* cs = is_v ? c.v_stride : c.k_stride;
      const int64_t off = outer * cs[0] + row * cs[1] + h * cs[2] + at * kPer;
      const void* base = is_v ? c.v : c.k;
      if constexpr (!kQuant) {
        raw[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(base) + off);
      } else {
        const int8_t* src = static_cast<const int8_t*>(base) + off;
        if constexpr (kPer == 8) {
          const uint2 x = *reinterpret_cast<const uint2*>(src);
          raw[i].x = x.x;
          raw[i].y = x.y;
        } else {
          raw[i].x = *reinterpret_cast<const uint32_t*>(src);
        }
        const int64_t* ss = is_v ? c.vs_stride : c.ks_stride;
        scale[i] = (is_v ? c.vs : c.ks)[outer * ss[0] + row * ss[1] + h * ss[2]];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int slot = slot0 + i * kRows + sub;
    if (slot >= slots) continue;
    const bool is_v = slot >= c.heads_kv;
    const int h = is_v ? slot - c.heads_kv : slot;
    uint4 out = raw[i];
    if constexpr (kQuant) {
      const int8_t* q = reinterpret_cast<const int8_t*>(&raw[i]);
      T* e = reinterpret_cast<T*>(&out);
#pragma unroll
      for (int j = 0; j < kPer; ++j) e[j] = from_float<T>(static_cast<float>(q[j]) * scale[i]);
    }
    const int64_t off = is_v ? t * r.v_stride[0] + h * r.v_stride[1]
                             : t * r.k_stride[0] + h * r.k_stride[1];
    *(reinterpret_cast<uint4*>(is_v ? r.v : r.k) + (off + at * kPer) / kPer) = out;
  }
}

// Rows a warp handles per lane: one for calls of few tokens, whose latency is what counts (more
// warps, each with one load), four for many (more bytes in flight per warp).
constexpr int kManyTokens = 512;

template <typename T, int D, bool kQuant>
int launch(const KvView& c, const RowsView& r, bool append, cudaStream_t stream) {
  constexpr int kRows = 32 / (D * static_cast<int>(sizeof(T)) / 16);
  const int iter = r.ragged.rows >= kManyTokens ? 4 : 1;
  const int per_token = (2 * c.heads_kv + kRows * iter - 1) / (kRows * iter);
  const int64_t warps = static_cast<int64_t>(r.ragged.rows) * per_token;
  const int64_t blocks = (warps * 32 + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return fail(FLB_ERR_UNSUPPORTED, "problem too large for one launch");
  const unsigned grid = static_cast<unsigned>(blocks);
  if (append) {
    if (iter == 4)
      kv_append_kernel<T, D, kQuant, 4><<<grid, kThreads, 0, stream>>>(c, r);
    else
      kv_append_kernel<T, D, kQuant, 1><<<grid, kThreads, 0, stream>>>(c, r);
    return check_cuda(cudaGetLastError(), "kv_append_kernel launch");
  }
  if (iter == 4)
    kv_gather_kernel<T, D, kQuant, 4><<<grid, kThreads, 0, stream>>>(c, r);
  else
    kv_gather_kernel<T, D, kQuant, 1><<<grid, kThreads, 0, stream>>>(c, r);
  return check_cuda(cudaGetLastError(), "kv_gather_kernel launch");
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
