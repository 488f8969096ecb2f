// Rotation of new queries and keys by their positions, and the append of keys and values to a paged cache, in one pass:
// every row is read once and written once (the rotated key goes straight into its page).
//
// A row of D values is handled by D/16 lanes, 16 values each: two 16-byte chunks that hold both halves of 8 rotation
// pairs (chunk c and chunk c + rotary_dim/16 when the pairs are (i, i + rotary_dim/2); two neighbouring chunks when they
// are (2i, 2i+1)). So a lane needs no other lane's values, and rotating in place is safe. A warp works on one token: its
// lanes keep their 8 cosines and sines in registers over U row groups of 32 / (D/16) heads.
// Bound: HBM; tokens * ((2 heads + 2 kv_heads) * D * 2 + 2 kv_heads * D * cache element) bytes. 23262 tokens, 32 / 8 heads of
// 128 in bf16: 91.5 us = 6.4 TB/s, 0.97 of the measured copy rate. Four row groups per warp: its look-ups and angles are
// shared by 16 rows of 128; rows are loaded ahead of the look-ups (131 us with each row loaded in its turn).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include "common.cuh"
#include "host_common.h"

namespace tb200 {

static constexpr int APP_WARPS = 8;

struct AppendParams {
  tb200_kv_append_args a;
  int rows;             // rows of one token: heads (0 without q) + 2 kv_heads
  int tasks_per_token;  // warps per token
};

template <bool F16>
__device__ __forceinline__ void widen8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <bool F16>
__device__ __forceinline__ uint4 narrow8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = F16 ? pack_f16x2(x[2 * i], x[2 * i + 1]) : pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// value / scale, round to nearest even, saturating at +-448 (NaN stays NaN)
__device__ __forceinline__ uint2 narrow8_e4m3(const float (&x)[8], float scale) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * i + 1] / scale), "f"(x[4 * i] / scale));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * i + 3] / scale), "f"(x[4 * i + 2] / scale));
    w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// Whole warp: the largest b in [0, n) with cu[b] <= t, or -1. 32 probes a step: two steps for up to 1024 sequences.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int n, int t, int lane) {
  int lo = 0, end = n;
  while (end - lo > 0) {
    const int step = (end - lo + 31) >> 5;
    const int i = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, i < end && cu[min(i, n - 1)] <= t);
    const int c = __popc(below);
    if (c == 0) return -1;
    lo += (c - 1) * step;
    end = min(end, lo + step);
    if (step == 1) break;
  }
  return lo;
}

template <int D, bool F16, bool C8, int U>
__global__ void __launch_bounds__(APP_WARPS * 32) kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = D / 16, RPW = 32 / LPR;
  const tb200_kv_append_args& a = p.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const uint32_t gw = blockIdx.x * APP_WARPS + (threadIdx.x >> 5);
  const uint32_t t = gw / (uint32_t)p.tasks_per_token;
  if (t >= (uint32_t)a.tokens) return;
  const int row0 = (int)(gw - t * p.tasks_per_token) * (RPW * U) + lane / LPR;
  const int n_q = a.q ? (int)a.heads : 0, n_kv = (int)a.kv_heads;

  // ---- this lane's two chunks of 8 columns
  const int item = lane % LPR, rot = a.cos ? a.rotary_dim : 0;
  const bool turns = item * 16 < rot;
  const bool halves = turns && !a.interleaved;
  const int c0 = halves ? item * 8 : item * 16;
  const int c1 = halves ? c0 + rot / 2 : c0 + 8;

  // ---- all rows first: where they go takes a chain of look-ups
  uint4 w0[U], w1[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * RPW;
    w0[u] = w1[u] = make_uint4(0, 0, 0, 0);
    if (row < p.rows) {
      const uint16_t* src = row < n_q ? (const uint16_t*)a.q + t * a.q_stride_tok + row * a.q_stride_head
                            : row < n_q + n_kv ? (const uint16_t*)a.k + t * a.k_stride_tok + (row - n_q) * a.k_stride_head
                                               : (const uint16_t*)a.v + t * a.v_stride_tok + (row - n_q - n_kv) * a.v_stride_head;
      w0[u] = *reinterpret_cast<const uint4*>(src + c0);
      w1[u] = *reinterpret_cast<const uint4*>(src + c1);
    }
  }

  // ---- the token's sequence, position, table row and page
  int b = (int)t;
  long long at = 1;  // rows from this one to the end of its sequence
  if (a.cu_seqlens) {
    b = find_sequence(a.cu_seqlens, (int)a.batch, (int)t, lane);
    if (b < 0) return;
    const int end = a.cu_seqlens[b + 1];
    if ((int)t >= end) return;  // behind the last sequence
    at = (long long)end - t;
  }
  const long long position = a.seq_lens[b] - at;
  const int pos = position >= 0 ? (int)position : -1;
  const int slot = pos >= 0 ? pos / a.page_size : -1;
  const bool valid = pos >= 0 && slot < a.max_pages && (!a.cos || pos < a.n_positions);
  int64_t page = -1;
  if (valid) page = a.page_table[b * a.table_stride + slot];
  const bool cached = page >= 0 && page < a.n_pages;
  const int in_page = valid ? pos - slot * a.page_size : 0;
  float cs[8], sn[8];  // the angles of this lane's 8 pairs
  if (turns && valid) {
    const float4* cr = reinterpret_cast<const float4*>(a.cos + pos * a.rot_stride + item * 8);
    const float4* sr = reinterpret_cast<const float4*>(a.sin + pos * a.rot_stride + item * 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = cr[i], s = sr[i];
      cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
      sn[4 * i] = s.x, sn[4 * i + 1] = s.y, sn[4 * i + 2] = s.z, sn[4 * i + 3] = s.w;
    }
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int row = row0 + u * RPW;
    if (row >= p.rows) break;
    const int which = row < n_q ? 0 : row < n_q + n_kv ? 1 : 2;
    const int h = which == 0 ? row : which == 1 ? row - n_q : row - n_q - n_kv;
    if (!valid) w0[u] = w1[u] = make_uint4(0, 0, 0, 0);
    float x[8], y[8];
    widen8<F16>(w0[u], x);
    widen8<F16>(w1[u], y);
    if (which < 2 && turns && valid) {
      if (halves) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xr = x[i] * cs[i] - y[i] * sn[i];
          y[i] = y[i] * cs[i] + x[i] * sn[i];
          x[i] = xr;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float r = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
          x[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
          x[2 * i] = r;
          r = y[2 * i] * cs[4 + i] - y[2 * i + 1] * sn[4 + i];
          y[2 * i + 1] = y[2 * i + 1] * cs[4 + i] + y[2 * i] * sn[4 + i];
          y[2 * i] = r;
        }
      }
      w0[u] = narrow8<F16>(x);
      w1[u] = narrow8<F16>(y);
    }
    uint16_t* packed = which == 0                ? (uint16_t*)a.q_out + t * a.qo_stride_tok + h * a.qo_stride_head
                       : which == 1 && a.k_out ? (uint16_t*)a.k_out + t * a.ko_stride_tok + h * a.ko_stride_head
                                                 : nullptr;
    if (packed) {
      *reinterpret_cast<uint4*>(packed + c0) = w0[u];
      *reinterpret_cast<uint4*>(packed + c1) = w1[u];
    }
    if (which > 0 && cached) {
      const int64_t at = which == 1
                             ? page * a.kc_stride_page + in_page * a.kc_stride_tok + h * a.kc_stride_head
                             : page * a.vc_stride_page + in_page * a.vc_stride_tok + h * a.vc_stride_head;
      void* pool = which == 1 ? a.k_cache : a.v_cache;
      if (C8) {
        const float* sc = which == 1 ? a.k_scale : a.v_scale;
        const float scale = sc[(which == 1 ? a.k_scale_n : a.v_scale_n) > 1 ? h : 0];
        uint8_t* dst = (uint8_t*)pool + at;
        *reinterpret_cast<uint2*>(dst + c0) = narrow8_e4m3(x, scale);
        *reinterpret_cast<uint2*>(dst + c1) = narrow8_e4m3(y, scale);
      } else {
        uint16_t* dst = (uint16_t*)pool + at;
        *reinterpret_cast<uint4*>(dst + c0) = w0[u];
        *reinterpret_cast<uint4*>(dst + c1) = w1[u];
      }
    }
  }
}

template <int D, int U>
static int launch_append(const AppendParams& p, cudaStream_t stream) {
  const bool f16 = p.a.dtype == TB200_F16, c8 = p.a.cache_dtype == TB200_E4M3;
  auto kfn = f16 ? (c8 ? kv_append_kernel<D, true, true, U> : kv_append_kernel<D, true, false, U>)
                 : (c8 ? kv_append_kernel<D, false, true, U> : kv_append_kernel<D, false, false, U>);
  const int64_t blocks = (p.a.tokens * p.tasks_per_token + APP_WARPS - 1) / APP_WARPS;
  if (blocks * APP_WARPS > INT32_MAX) return TB200_ERR_UNSUPPORTED;
  return cuda_err(launch_overlapped(kfn, dim3((unsigned)blocks), APP_WARPS * 32, 0, stream, p));
}

}  // namespace tb200

using namespace tb200;

static bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

extern "C" int tb200_kv_append(const tb200_kv_append_args* a, void* stream_) {
  if (!a) return TB200_ERR_BAD_ARG;
  if (a->tokens < 0 || a->batch < 0 || a->heads < 0 || a->kv_heads < 1 || a->n_pages < 0 || a->max_pages < 0 ||
      a->page_size < 1)
    return TB200_ERR_BAD_ARG;
  if (!a->cu_seqlens && a->tokens != a->batch) return TB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return TB200_ERR_UNSUPPORTED;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  const bool c8 = a->cache_dtype == TB200_E4M3;
  if (!c8 && a->cache_dtype != a->dtype) return TB200_ERR_UNSUPPORTED;
  if (c8 && ((a->k_scale_n != 1 && a->k_scale_n != a->kv_heads) || (a->v_scale_n != 1 && a->v_scale_n != a->kv_heads)))
    return TB200_ERR_BAD_ARG;
  if ((a->q != nullptr) != (a->q_out != nullptr) || (a->cos != nullptr) != (a->sin != nullptr)) return TB200_ERR_BAD_ARG;
  if (a->cos && (a->rotary_dim < 16 || a->rotary_dim > a->head_dim || a->rotary_dim % 16 || a->n_positions < 0))
    return TB200_ERR_BAD_ARG;
  if (a->tokens > INT32_MAX || a->batch > INT32_MAX - 1 || a->heads > (1 << 20) || a->kv_heads > (1 << 20))
    return TB200_ERR_UNSUPPORTED;
  if (misaligned(a->q, 16) || misaligned(a->k, 16) || misaligned(a->v, 16) || misaligned(a->q_out, 16) ||
      misaligned(a->k_out, 16) || misaligned(a->cos, 16) || misaligned(a->sin, 16) || a->rot_stride % 4 || misaligned(a->k_cache, c8 ? 8 : 16) || misaligned(a->v_cache, c8 ? 8 : 16))
    return TB200_ERR_BAD_ARG;
  const int64_t strides[] = {a->q_stride_tok,  a->q_stride_head,  a->k_stride_tok,  a->k_stride_head,
                             a->v_stride_tok,  a->v_stride_head,  a->qo_stride_tok, a->qo_stride_head,
                             a->ko_stride_tok, a->ko_stride_head, a->kc_stride_page, a->kc_stride_tok,
                             a->kc_stride_head, a->vc_stride_page, a->vc_stride_tok, a->vc_stride_head};
  for (int64_t s : strides)
    if (s % 8) return TB200_ERR_BAD_ARG;
  if (a->tokens == 0 || a->batch == 0) return TB200_OK;
  if (!a->k || !a->v || !a->seq_lens || (a->n_pages > 0 && (!a->k_cache || !a->v_cache)) ||
      (a->max_pages > 0 && !a->page_table) || (c8 && (!a->k_scale || !a->v_scale)))
    return TB200_ERR_BAD_ARG;

  AppendParams p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.rows = (a->q ? (int)a->heads : 0) + 2 * (int)a->kv_heads;
  constexpr int U = 4;
  const int per_warp = 32 / (a->head_dim / 16) * U;
  p.tasks_per_token = (p.rows + per_warp - 1) / per_warp;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return a->head_dim == 64 ? launch_append<64, U>(p, stream)
         : a->head_dim == 128 ? launch_append<128, U>(p, stream) : launch_append<256, U>(p, stream);
}
