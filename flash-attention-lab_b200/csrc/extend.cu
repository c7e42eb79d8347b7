// Attention of new tokens over a cache that already holds their K and V (flb_extend_fwd).
// A warp owns one (row, head): its lanes hold D / 32 values of q and o each, and it walks the keys
// the row sees with an online softmax in fp32.
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

struct ExtendArgs {
  const void* q;
  void* o;
  float* lse;
  int64_t q_stride[2], o_stride[2];   // row, head
  const int32_t* seq_lens;
  Ragged ragged;
  int heads, group, causal;
  float scale_log2;
};

template <typename T, typename C, int D>
__global__ void __launch_bounds__(128) extend_kernel(const __grid_constant__ KvView c,
                                                     const __grid_constant__ ExtendArgs a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int t = static_cast<int>(w / a.heads);
  const int h = static_cast<int>(w - static_cast<int64_t>(t) * a.heads);
  if (t >= a.ragged.rows) return;
  const int hkv = h / a.group;
  int b, first, count, seen = 0;
  if (find_sequence(a.ragged, t, lane, b, first, count)) {
    const int len = min(max(__ldg(a.seq_lens + b), 0), c.max_seqlen);
    seen = a.causal ? min(len, len - count + (t - first) + 1) : len;
  }
  float q[kPer], o[kPer], m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(a.q) + t * a.q_stride[0] + h * a.q_stride[1];
  for (int i = 0; i < kPer; ++i) {
    q[i] = static_cast<float>(qp[lane * kPer + i]);
    o[i] = 0.f;
  }
  for (int j = 0; j < seen; ++j) {
    int64_t outer, row;
    const bool in = c.locate(b, j, outer, row);   // keys of a bad block read as zeros
    float s = 0.f, vs = 1.f;
    if (in) {
      const C* kp = static_cast<const C*>(c.k) + outer * c.k_stride[0] + row * c.k_stride[1] +
                    hkv * c.k_stride[2];
      for (int i = 0; i < kPer; ++i) s += q[i] * static_cast<float>(kp[lane * kPer + i]);
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      s *= a.scale_log2;
      if (c.ks != nullptr) {
        s *= c.ks[outer * c.ks_stride[0] + row * c.ks_stride[1] + hkv * c.ks_stride[2]];
        vs = c.vs[outer * c.vs_stride[0] + row * c.vs_stride[1] + hkv * c.vs_stride[2]];
      }
    }
    const float m_new = fmaxf(m, s), f = exp2f(m - m_new), p = exp2f(s - m_new);
    m = m_new;
    l = l * f + p;
    const C* vp = static_cast<const C*>(c.v) + outer * c.v_stride[0] + row * c.v_stride[1] +
                  hkv * c.v_stride[2];
    for (int i = 0; i < kPer; ++i)
      o[i] = o[i] * f + (in ? p * vs * static_cast<float>(vp[lane * kPer + i]) : 0.f);
  }
  T* op = static_cast<T*>(a.o) + t * a.o_stride[0] + h * a.o_stride[1];
  for (int i = 0; i < kPer; ++i) {
    const float x = seen > 0 ? o[i] / l : 0.f;
    if constexpr (std::is_same<T, __half>::value) {
      op[lane * kPer + i] = __float2half_rn(x);
    } else {
      op[lane * kPer + i] = __float2bfloat16_rn(x);
    }
  }
  if (lane == 0)
    a.lse[static_cast<int64_t>(t) * a.heads + h] =
        seen > 0 ? m * 0.69314718055994530942f + logf(l) : -INFINITY;
}

template <typename T, typename C>
int launch(const flb_kv_cache* c, const KvView& cv, const ExtendArgs& a, cudaStream_t stream) {
  const int64_t warps = static_cast<int64_t>(a.ragged.rows) * a.heads;
  const unsigned grid = static_cast<unsigned>((warps + 3) / 4);
  if (c->head_dim == 128)
    extend_kernel<T, C, 128><<<grid, 128, 0, stream>>>(cv, a);
  else
    extend_kernel<T, C, 64><<<grid, 128, 0, stream>>>(cv, a);
  return check_cuda(cudaGetLastError(), "extend_kernel launch");
}

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
  if (p->heads / c->heads_kv > 128)
    return fail(FLB_ERR_UNSUPPORTED, "more than 128 query heads per KV head");
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
  const View4 qv{p->q, {1, p->rows, p->heads, c->head_dim},
                 {0, p->q_row_stride, p->q_head_stride, 1}, 2};
  const View4 ov{p->o, {1, p->rows, p->heads, c->head_dim},
                 {0, p->o_row_stride, p->o_head_stride, 1}, 2};
  if (!rows_16b_aligned(qv))
    return fail(FLB_ERR_MISALIGNED, "q must have 16-byte aligned rows (data pointer and strides)");
  if (!rows_16b_aligned(ov))
    return fail(FLB_ERR_MISALIGNED, "o must have 16-byte aligned rows (data pointer and strides)");
  if (static_cast<int64_t>(p->rows) * p->heads > 0x7fffffffLL)
    return fail(FLB_ERR_UNSUPPORTED, "problem too large for one launch");
  return FLB_OK;
}

}  // namespace
}  // namespace flb

using namespace flb;

extern "C" size_t flb_extend_workspace_bytes(int32_t, int32_t, int32_t, int32_t, int32_t) {
  return 0;
}

extern "C" int flb_extend_fwd(const flb_kv_cache* c, const flb_extend_params* p,
                              flb_stream_t stream_) {
  clear_error();
  if (int st = validate(c, p)) return st;
  if (int st = current_device_info(nullptr, nullptr, nullptr, nullptr)) return st;
  ExtendArgs a{};
  a.q = p->q;
  a.o = p->o;
  a.lse = p->lse;
  a.q_stride[0] = p->q_row_stride;
  a.q_stride[1] = p->q_head_stride;
  a.o_stride[0] = p->o_row_stride;
  a.o_stride[1] = p->o_head_stride;
  a.seq_lens = p->seq_lens;
  a.ragged = Ragged{p->cu_seqlens, p->rows, p->rows_per_seq, c->batch};
  a.heads = p->heads;
  a.group = p->heads / c->heads_kv;
  a.causal = p->causal ? 1 : 0;
  a.scale_log2 = static_cast<float>(static_cast<double>(p->softmax_scale) * 1.4426950408889634);
  const KvView cv = kv_view(c);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (p->dtype == FLB_BF16)
    return c->dtype == FLB_INT8 ? launch<__nv_bfloat16, int8_t>(c, cv, a, stream)
                                : launch<__nv_bfloat16, __nv_bfloat16>(c, cv, a, stream);
  return c->dtype == FLB_INT8 ? launch<__half, int8_t>(c, cv, a, stream)
                              : launch<__half, __half>(c, cv, a, stream);
}
