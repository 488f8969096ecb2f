// Attention of one new token per sequence over a paged KV cache.
//
// One warp per (sequence, query head): lane l holds columns l * D/32 .. of the query, the accumulator and the key /
// value row in flight; the score is a butterfly sum, the softmax is kept online (running maximum and sum in fp32).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include "attention_common.cuh"
#include "common.cuh"
#include "host_common.h"

namespace tb200 {

struct DecodeParams {
  tb200_attention_decode_args a;
  float scale_log2;
};

template <int D, bool F16, bool C8>
__global__ void __launch_bounds__(128) attention_decode_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int V = D / 32;
  const tb200_attention_decode_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.batch * a.heads) return;
  const int64_t b = row / a.heads, h = row % a.heads, kvh = h / (a.heads / a.kv_heads);
  auto widen = [](uint16_t v) { return F16 ? __half2float(__ushort_as_half(v)) : __uint_as_float((uint32_t)v << 16); };
  auto cached = [&](const void* pool, int64_t at) {
    if (!C8) return widen(((const uint16_t*)pool)[at]);
    uint32_t w;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(w) : "h"((uint16_t)((const uint8_t*)pool)[at]));
    return __half2float(__ushort_as_half((uint16_t)w));
  };
  float q[V], o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    q[i] = widen(((const uint16_t*)a.q)[b * a.q_stride_b + h * a.q_stride_head + lane * V + i]);
    o[i] = 0.f;
  }
  float scale = p.scale_log2, v_scale = 1.f;
  if (C8) {
    scale *= a.k_scale[a.k_scale_n > 1 ? kvh : 0];
    v_scale = a.v_scale[a.v_scale_n > 1 ? kvh : 0];
  }
  const int64_t len = min(max((int64_t)a.seq_lens[b], (int64_t)0), a.max_pages * a.page_size);
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < len; ++j) {
    const int64_t page = a.page_table[b * a.table_stride + j / a.page_size], in_page = j % a.page_size;
    const bool there = page >= 0 && page < a.n_pages;
    const int64_t ka = page * a.kc_stride_page + in_page * a.kc_stride_tok + kvh * a.kc_stride_head + lane * V;
    const int64_t va = page * a.vc_stride_page + in_page * a.vc_stride_tok + kvh * a.vc_stride_head + lane * V;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += there ? q[i] * cached(a.k_cache, ka + i) : 0.f;
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= scale;
    const float m_new = fmaxf(m, s), m_ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m - m_ref), e = fast_exp2(s - m_ref);
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = o[i] * alpha + (there ? e * cached(a.v_cache, va + i) : 0.f);
    m = m_new;
  }
  const float inv = l > 0.f ? v_scale / l : 0.f;
  uint16_t* out = (uint16_t*)a.o + b * a.o_stride_b + h * a.o_stride_head + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i)
    out[i] = F16 ? __half_as_ushort(__float2half_rn(o[i] * inv)) : __bfloat16_as_ushort(__float2bfloat16_rn(o[i] * inv));
  if (a.lse && lane == 0) a.lse[row] = l > 0.f ? m + log2f(l) : -INFINITY;
}

template <int D>
static int launch_decode(const DecodeParams& p, cudaStream_t stream) {
  const bool f16 = p.a.dtype == TB200_F16, c8 = p.a.cache_dtype == TB200_E4M3;
  auto kfn = f16 ? (c8 ? attention_decode_kernel<D, true, true> : attention_decode_kernel<D, true, false>)
                 : (c8 ? attention_decode_kernel<D, false, true> : attention_decode_kernel<D, false, false>);
  const int64_t rows = p.a.batch * p.a.heads;
  kfn<<<(unsigned)((rows + 3) / 4), 128, 0, stream>>>(p);
  return cuda_err(cudaGetLastError());
}

}  // namespace tb200

using namespace tb200;

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

extern "C" size_t tb200_attention_decode_workspace_bytes(const tb200_attention_decode_args*) { return 0; }

extern "C" int tb200_attention_decode(const tb200_attention_decode_args* a, void* stream_) {
  if (!a) return TB200_ERR_BAD_ARG;
  if (a->batch < 0 || a->heads < 0 || a->kv_heads < 1 || a->heads % a->kv_heads || a->n_pages < 0 || a->max_pages < 0 ||
      a->page_size < 1)
    return TB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return TB200_ERR_UNSUPPORTED;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  const bool c8 = a->cache_dtype == TB200_E4M3;
  if (!c8 && a->cache_dtype != a->dtype) return TB200_ERR_UNSUPPORTED;
  if (c8 && ((a->k_scale_n != 1 && a->k_scale_n != a->kv_heads) || (a->v_scale_n != 1 && a->v_scale_n != a->kv_heads)))
    return TB200_ERR_BAD_ARG;
  if (!(a->sm_scale > 0.f)) return TB200_ERR_BAD_ARG;
  if (off16(a->q) || off16(a->o) || off16(a->k_cache) || off16(a->v_cache)) return TB200_ERR_BAD_ARG;
  const int64_t rows[] = {a->q_stride_b, a->q_stride_head, a->o_stride_b, a->o_stride_head};
  for (int64_t s : rows)
    if (s % 8) return TB200_ERR_BAD_ARG;
  const int64_t pools[] = {a->kc_stride_page, a->kc_stride_tok, a->kc_stride_head,
                           a->vc_stride_page, a->vc_stride_tok, a->vc_stride_head};
  for (int64_t s : pools)
    if (s % (c8 ? 16 : 8)) return TB200_ERR_BAD_ARG;
  if (a->batch > INT32_MAX || a->heads > (1 << 16) || a->batch * a->heads > INT32_MAX || a->max_pages > INT32_MAX ||
      a->max_pages * a->page_size > (1 << 30))
    return TB200_ERR_UNSUPPORTED;
  if (a->batch == 0 || a->heads == 0) return TB200_OK;
  if (!a->q || !a->o || !a->seq_lens || (a->n_pages > 0 && (!a->k_cache || !a->v_cache)) ||
      (a->max_pages > 0 && !a->page_table) || (c8 && (!a->k_scale || !a->v_scale)))
    return TB200_ERR_BAD_ARG;
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return a->head_dim == 64 ? launch_decode<64>(p, stream)
         : a->head_dim == 128 ? launch_decode<128>(p, stream) : launch_decode<256>(p, stream);
}
