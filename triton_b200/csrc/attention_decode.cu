// Attention of one new token per sequence over a paged KV cache.
//
// The work is every (sequence, kv head, group of up to 8 NT query heads) times its tiles of KS keys, laid out as one line of
// tiles; each warp takes an equal piece of the line, whatever the lengths are, and runs on its own: a stretch (the tiles of one
// sequence and head group) that lies in its piece is written out from its registers. Parts of stretches that are cut at
// the borders of pieces are (unnormalised accumulator, maximum, sum); those inside a CTA are merged through shared memory at
// the CTA's end, those between CTAs go to the workspace and a second small kernel joins them, in the order of the line (no
// atomics: equal inputs give equal bits).
//
// A warp keeps a ring of steps in flight by 16-byte cp.async (keys behind the end and pages outside the pool are filled with
// zeros without an access). The products run on the tensor cores with the keys as the long side: S^T [16 keys, 8 heads] =
// K Q^T and O^T [16 columns, 8 heads] += V^T P^T by mma.m16n8k16, so a group of up to 8 heads fills the 8-wide side whatever
// its size. tcgen05 has no use here: its 128-row tile would be filled by 8 heads, and the kernel is bound by reading K and V.
// Bound: HBM. 2 sequences of 374000 tokens, 64 / 8 heads of 128 in bf16: 459 us = 6.7 TB/s; 64 sequences of 9000 in e4m3:
// 199 us = 6.0 TB/s; 48 sequences up to 6000 tokens, 32 / 8 heads: 45 us, of which 23 are reading and the rest start-up,
// merging and joining.
// e4m3 pools are widened to float16 in registers (exact); queries are then brought to [1, 2) by a power of two per head
// first, so that they fit. P is rounded to the type of V (float16 for e4m3), everything else is kept in 32 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>

#include "attention_common.cuh"
#include "common.cuh"
#include "host_common.h"

namespace tb200 {

static constexpr int DEC_WARPS = 4;
static constexpr float DEC_RESCALE_THRESHOLD = 8.0f;  // the accumulator is rescaled when a maximum grew by more than 2^8

enum DecKind { DEC_BF16 = 0, DEC_F16 = 1, DEC_E4M3 = 2 };

// One CTA's first stretch: the line positions [s, e) of the whole stretch, for the join.
struct DecMeta {
  int b, hg, s, e;
};

struct DecodeParams {
  tb200_attention_decode_args a;
  float scale_log2;
  int group, groups_per_kv, hgs;  // query heads per kv head; head groups per kv head; head groups in all
  int max_len;
  uint32_t page_mul, page_shift;  // n / page_size = umulhi(2 n, page_mul) >> page_shift for n < 2^30
  long long k_page, k_tok, k_head, v_page, v_tok, v_head;  // strides of the pools in bytes
  float* warp_o;                  // [CTA][warp][heads of a group][D]: parts cut at the start of a warp's piece
  float* part_o;                  // [CTA][2][heads of a group][D]: a stretch cut at the CTA's start (0) or end (1)
  float2* part_ml;                // [CTA][2][heads of a group]
  DecMeta* meta;                  // [CTA]
  int* per;                       // tiles per CTA
};

template <int D, int KIND, int NT>
struct DecCfg {
  static constexpr int ESZ = KIND == DEC_E4M3 ? 1 : 2;
  static constexpr int ROW = D * ESZ;                    // bytes of a K or V row
  static constexpr int CH = ROW / 16;                    // 16-byte chunks of it
  static constexpr int KS = ROW >= 256 ? 16 : 32;        // keys per step
  static constexpr int STAGE = 2 * KS * ROW;             // K then V
  static constexpr int CTAS = D == 256 ? 1 : 2;          // per SM; together they keep up to 192 KB in flight
  static constexpr int STAGES = 196608 / (CTAS * DEC_WARPS * STAGE);
  static constexpr int NH = 8 * NT;
  static constexpr int RING = DEC_WARPS * STAGES * STAGE;
  static constexpr int PARTS = 2 * DEC_WARPS;            // of its warps' pieces, a cut stretch at each end
  static constexpr int HEAD = NH * D * 4;                // bytes of a part's accumulator
  static constexpr int LIMIT = 233472 / CTAS - 1024;
  // A part that is cut at a piece's end takes the place of the warp's ring, which is empty by then; one that is cut at its
  // start has shared memory of its own where that fits, else it goes through the workspace.
  static constexpr int SCRATCH = DEC_WARPS * (2 * 4 + 16);  // of the kernel's head: sums and starts of its warps
  static constexpr bool HEAD_SMEM = RING + DEC_WARPS * HEAD + PARTS * (NH * 8 + 16) + SCRATCH <= LIMIT;
  static constexpr int HEADS = HEAD_SMEM ? DEC_WARPS * HEAD : 0;
  static constexpr int SMEM = RING + HEADS + PARTS * (NH * 8 + 16) + SCRATCH;
  static_assert(HEAD <= STAGES * STAGE, "a part fits the ring of a warp");
};

__device__ __forceinline__ void dec_cp16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void dec_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void dec_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t dec_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool BF>
__device__ __forceinline__ void dec_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t dec_widen_e4m3(uint32_t two) {  // the low two bytes -> two halves
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ float2 dec_unpack(uint32_t w, bool f16) {
  return f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w))
             : make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ int dec_len(const DecodeParams& p, int b) { return min(max(p.a.seq_lens[b], 0), p.max_len); }

__device__ __forceinline__ uint16_t* dec_out(const DecodeParams& p, int b, int h) {
  return (uint16_t*)p.a.o + (long long)b * p.a.o_stride_b + (long long)h * p.a.o_stride_head;
}
__device__ __forceinline__ uint32_t dec_pack_out(const DecodeParams& p, float x, float y) {
  return p.a.dtype == TB200_F16 ? pack_f16x2(x, y) : pack_bf16x2(x, y);
}

// A stretch that a part in shared memory belongs to.
struct DecPart {
  int s;  // where the stretch begins on the line; -1: no part
  int b, hg, nt;
};

template <int D, int KIND, int NT>
__global__ void __launch_bounds__(DEC_WARPS * 32, DecCfg<D, KIND, NT>::CTAS)
    attention_decode_kernel(const __grid_constant__ DecodeParams p) {
  using C = DecCfg<D, KIND, NT>;
  constexpr int KT = C::KS / 16, KSTEPS = D / 16, STAGES = C::STAGES, NH = C::NH, RPI = 32 / C::CH;
  constexpr bool BF = KIND == DEC_BF16;
  extern __shared__ __align__(128) uint8_t smem[];
  float2* part_ml = reinterpret_cast<float2*>(smem + C::RING + C::HEADS);                  // [part][head]
  DecPart* parts = reinterpret_cast<DecPart*>(smem + C::RING + C::HEADS + C::PARTS * NH * 8);  // [part]
  int* sh_sum = reinterpret_cast<int*>(parts + C::PARTS);                                  // [warp], room for two each
  int4* sh_at = reinterpret_cast<int4*>(sh_sum + 2 * DEC_WARPS);  // [warp] where its piece begins: sequence, length, head group, tile
  const tb200_attention_decode_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int batch = (int)a.batch;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // what ran before: it may still be ending while this starts
  asm volatile("griddepcontrol.launch_dependents;");

  // ---- this warp's piece of the line (its length fits 32 bits: the host has seen to it)
  const int chunk = (batch + DEC_WARPS * 32 - 1) / (DEC_WARPS * 32);
  const int b_lo = min((int)threadIdx.x * chunk, batch), b_hi = min(b_lo + chunk, batch);
  auto tiles_of = [](int len) { return (len + C::KS - 1) / C::KS; };
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += tiles_of(dec_len(p, b)) * p.hgs;
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) sh_sum[warp] = upto;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < DEC_WARPS; ++w) {
    if (w < warp) upto += sh_sum[w];
    total += sh_sum[w];
  }
  const uint32_t n_warps = gridDim.x * DEC_WARPS;
  const int per = (int)max(((uint32_t)total + n_warps - 1) / n_warps, 1u);  // tiles of a warp
  const int cta_first = (int)min((long long)per * DEC_WARPS * blockIdx.x, (long long)total);
  const int cta_last = min(cta_first + per * DEC_WARPS, total);
  for (int w = 0; w < DEC_WARPS; ++w) {
    const int target = cta_first + per * w;
    if (target < upto && upto - mine <= target) {
      int at = upto - mine;
      for (int b = b_lo; b < b_hi; ++b) {
        const int len = dec_len(p, b), nt = tiles_of(len), rem = target - at;
        if (rem < nt * p.hgs) {
          const int hg = rem / nt;
          sh_at[w] = make_int4(b, len, hg, rem - hg * nt);
          break;
        }
        at += nt * p.hgs;
      }
    }
  }
  __syncthreads();
  const int first = cta_first + per * warp, last = min(first + per, cta_last);
  const bool works = first < last;

  // ---- positions on the line: one runs ahead for the loads, one for the products
  struct At {
    int b, hg, t, nt, len;
    int next;  // the length of sequence b + 1, read ahead
  };
  auto enter = [&](At& x, int b, int len) {
    x.b = b;
    x.len = len;
    x.nt = tiles_of(len);
    x.next = b + 1 < batch ? dec_len(p, b + 1) : 0;
  };
  auto next_stretch = [&](At& x) {
    x.t = 0;
    if (++x.hg < p.hgs) return;
    x.hg = 0;
    int b = x.b + 1, len = x.next;
    while (len == 0 && b + 1 < batch) len = dec_len(p, ++b);
    if (b < batch) enter(x, b, len);
  };
  At ld = {};
  if (works) {
    const int4 x = sh_at[warp];
    enter(ld, x.x, x.y);
    ld.hg = x.z;
    ld.t = x.w;
  }
  At cur = ld;
  if (lane < 2) parts[2 * warp + lane].s = -1;
  auto part_o = [&](int part) {
    if (part & 1) return reinterpret_cast<float*>(smem + (part >> 1) * STAGES * C::STAGE);
    if (C::HEAD_SMEM) return reinterpret_cast<float*>(smem + C::RING + (part >> 1) * C::HEAD);
    return p.warp_o + ((long long)blockIdx.x * DEC_WARPS + (part >> 1)) * NH * D;
  };

  const uint32_t ring = smem_u32(smem) + warp * STAGES * C::STAGE;
  const bool page_steps = a.page_size % C::KS == 0;  // then a step's keys lie in one page
  const int row0 = lane / C::CH, col0 = lane % C::CH * 16;
  // Places of a step's rows: lane r looks up row r (page_steps: all lanes the step's first row). The page table passes
  // through a window of 64 entries in two registers, so a step finds its pages there without waiting for memory.
  int win_b = -1, win0 = 0, win_lo = -1, win_hi = -1;
  auto page_entry = [&](int slot) {
    return slot < (int)a.max_pages && (long long)slot * a.page_size < ld.len ? a.page_table[ld.b * a.table_stride + slot] : -1;
  };
  const uint8_t *k_at = nullptr, *v_at = nullptr;
  long long k_kvh = 0, v_kvh = 0;  // byte offsets of the kv head
  int rows = 0;                    // rows of the step that exist
  bool there = false;              // this lane's row (page_steps: the step) has a page
  auto enter_head = [&]() {
    const int kvh = ld.hg / p.groups_per_kv;
    k_kvh = kvh * p.k_head;
    v_kvh = kvh * p.v_head;
  };
  auto look_up = [&]() {
    const int key0 = ld.t * C::KS;
    rows = min(ld.len - key0, C::KS);
    there = false;
    auto slot_of = [&](int key) { return (int)(__umulhi((uint32_t)key * 2u, p.page_mul) >> p.page_shift); };
    const int first_slot = slot_of(key0);
    if (ld.b != win_b || first_slot < win0) {
      win_b = ld.b;
      win0 = first_slot;
      win_lo = page_entry(win0 + lane);
      win_hi = page_entry(win0 + 32 + lane);
    } else if (first_slot >= win0 + 32) {  // a step never moves on by more than 32 pages
      win0 += 32;
      win_lo = win_hi;
      win_hi = page_entry(win0 + 32 + lane);
    }
    const int r = page_steps ? 0 : lane % C::KS;
    const int key = key0 + r, slot = slot_of(key), in_page = key - slot * a.page_size;
    int page = __shfl_sync(0xffffffffu, win_lo, (slot - win0) & 31);
    if (!page_steps) {
      const int high = __shfl_sync(0xffffffffu, win_hi, (slot - win0) & 31);
      if (slot - win0 >= 32) page = high;
    }
    if (r < rows) {
      there = page >= 0 && page < (int)a.n_pages;
      k_at = (const uint8_t*)a.k_cache + page * p.k_page + in_page * p.k_tok + k_kvh;
      v_at = (const uint8_t*)a.v_cache + page * p.v_page + in_page * p.v_tok + v_kvh;
    }
  };
  // chunk c of row r goes to chunk c ^ (r % 8) (rows of 64 bytes: c ^ (r / 2 % 4)): eight rows at one column, which is
  // what ldmatrix reads, lie in different banks
  auto swizzle = [](int r) { return C::CH >= 8 ? (r & 7) << 4 : ((r >> 1) & 3) << 4; };
  auto issue = [&](int stage) {
    const uint32_t dst = ring + stage * C::STAGE + row0 * C::ROW;
    if (page_steps && there && rows == C::KS) {
      const uint8_t* kp = k_at + row0 * p.k_tok + col0;
      const uint8_t* vp = v_at + row0 * p.v_tok + col0;
      const long long k_step = RPI * p.k_tok, v_step = RPI * p.v_tok;
#pragma unroll
      for (int i = 0; i < C::KS / RPI; ++i) {
        const uint32_t to = dst + i * RPI * C::ROW + (col0 ^ swizzle(i * RPI + row0));
        dec_cp16(to, kp, true);
        dec_cp16(to + C::KS * C::ROW, vp, true);
        kp += k_step;
        vp += v_step;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < C::KS / RPI; ++i) {
      const int r = i * RPI + row0;
      const uint8_t *kp, *vp;
      bool ok = there;
      if (page_steps) {
        kp = k_at + r * p.k_tok;
        vp = v_at + r * p.v_tok;
      } else {
        kp = (const uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)k_at, r);
        vp = (const uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)v_at, r);
        ok = __shfl_sync(0xffffffffu, (int)there, r) != 0;
      }
      ok = ok && r < rows;
      const uint32_t to = dst + i * RPI * C::ROW + (col0 ^ swizzle(r));
      dec_cp16(to, ok ? kp + col0 : (const uint8_t*)a.k_cache, ok);
      dec_cp16(to + C::KS * C::ROW, ok ? vp + col0 : (const uint8_t*)a.v_cache, ok);
    }
  };
  int to_load = last - first;
  auto load_next = [&](int stage) {
    if (to_load > 0) {
      issue(stage);
      if (--to_load > 0) {
        if (++ld.t == ld.nt) {
          next_stretch(ld);
          enter_head();
        }
        look_up();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // ---- queries of the stretch ahead: the words as they are, and what they become
  uint32_t qf[NT][KSTEPS][2];
  int kvh = 0, head0 = 0, heads = 0;
  auto load_q = [&](const At& x) {
    kvh = x.hg / p.groups_per_kv;
    head0 = kvh * p.group + (x.hg - kvh * p.groups_per_kv) * NH;
    heads = min(NH, (kvh + 1) * p.group - head0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + lane / 4;
      const uint16_t* row = (const uint16_t*)a.q + x.b * a.q_stride_b + (head0 + h) * a.q_stride_head;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        qf[nt][k][0] = qf[nt][k][1] = 0u;
        if (h < heads) {
          if (KIND != DEC_E4M3) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(row + k * 16 + 2 * (lane & 3));
            qf[nt][k][0] = w[0];
            qf[nt][k][1] = w[4];
          } else {  // columns 4t .. 4t + 3 of each 16, the order in which ldmatrix hands out bytes
            const uint2 w = *reinterpret_cast<const uint2*>(row + k * 16 + 4 * (lane & 3));
            qf[nt][k][0] = w.x;
            qf[nt][k][1] = w.y;
          }
        }
      }
    }
  };
  float o[NT][KSTEPS][4], m[NT][2], l[NT][2], sc[NT][2];
  auto begin = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sc[nt][0] = sc[nt][1] = p.scale_log2;
      if (KIND == DEC_E4M3) {
        const bool f16 = a.dtype == TB200_F16;
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const float2 x = dec_unpack(qf[nt][k][0], f16), y = dec_unpack(qf[nt][k][1], f16);
          most = fmaxf(most, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const bool usual = most > 1e-30f && most < 1e30f;
        const int e = usual ? (int)((__float_as_uint(most) >> 23) & 0xff) - 127 : 0;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          const float2 x = dec_unpack(qf[nt][k][0], f16), y = dec_unpack(qf[nt][k][1], f16);
          qf[nt][k][0] = pack_f16x2(x.x * down, x.y * down);
          qf[nt][k][1] = pack_f16x2(y.x * down, y.y * down);
        }
        const float ks = p.scale_log2 * a.k_scale[a.k_scale_n > 1 ? kvh : 0];
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[nt][j] = ks * __shfl_sync(0xffffffffu, up, 4 * (2 * (lane & 3) + j));
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = -INFINITY;
        l[nt][j] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][k][i] = 0.f;
    }
  };
  if (works) {
    enter_head();
    look_up();
    load_q(cur);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load_next(s);
  }

  // ---- what nothing waits for: the join's view of this CTA, sequences without a key
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) *p.per = per * DEC_WARPS;
    p.meta[blockIdx.x] = DecMeta{works ? cur.b : -1, cur.hg, first - cur.t, first - cur.t + cur.nt};
  }
  for (int b = blockIdx.x; b < batch; b += gridDim.x) {
    if (dec_len(p, b) > 0) continue;
    for (int i = threadIdx.x; i < (int)a.heads * (D / 2); i += blockDim.x)
      reinterpret_cast<uint32_t*>(dec_out(p, b, i / (D / 2)))[i % (D / 2)] = 0u;
    if (a.lse)
      for (int h = threadIdx.x; h < (int)a.heads; h += blockDim.x) a.lse[(long long)b * a.heads + h] = -INFINITY;
  }

  // ---- the loop
  bool fresh = true;
  int stage = 0;
  for (int at = first; at < last; ++at) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    load_next(stage == 0 ? STAGES - 1 : stage - 1);
    if (fresh) begin();
    fresh = false;
    const int key0 = cur.t * C::KS;
    const uint32_t ks_base = ring + stage * C::STAGE, vs_base = ks_base + C::KS * C::ROW;
    // ---- scores
    float s[KT][NT][4];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kt][nt][i] = 0.f;
      const int r = kt * 16 + (lane & 15);
      const uint32_t row_at = ks_base + r * C::ROW;
      const int x = swizzle(r);
#pragma unroll
      for (int c = 0; c < C::CH / 2; ++c) {  // 32 bytes of the rows at a time
        uint32_t f[4];
        dec_ldsm(row_at + (((2 * c + (lane >> 4)) << 4) ^ x), f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (KIND != DEC_E4M3) {
            dec_mma<BF>(s[kt][nt], f[0], f[1], f[2], f[3], qf[nt][c][0], qf[nt][c][1]);
          } else {
            dec_mma<false>(s[kt][nt], dec_widen_e4m3(f[0]), dec_widen_e4m3(f[1]), dec_widen_e4m3(f[0] >> 16),
                           dec_widen_e4m3(f[1] >> 16), qf[nt][2 * c % KSTEPS][0], qf[nt][2 * c % KSTEPS][1]);
            dec_mma<false>(s[kt][nt], dec_widen_e4m3(f[2]), dec_widen_e4m3(f[3]), dec_widen_e4m3(f[2] >> 16),
                           dec_widen_e4m3(f[3] >> 16), qf[nt][(2 * c + 1) % KSTEPS][0], qf[nt][(2 * c + 1) % KSTEPS][1]);
          }
        }
      }
    }
    // ---- softmax: rows are keys (lane / 4 and 8 more), columns heads (2 (lane % 4) and the next)
    const bool ragged = key0 + C::KS > cur.len;
    float mx[NT][2];
    bool grew = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float& v = s[kt][nt][2 * u + j];
            v *= sc[nt][j];
            if (ragged && key0 + kt * 16 + u * 8 + lane / 4 >= cur.len) v = -INFINITY;
            t = fmaxf(t, v);
          }
        mx[nt][j] = t;
        grew = grew || t > m[nt][j] + DEC_RESCALE_THRESHOLD;
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float t = fmaxf(mx[nt][j], m[nt][j]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, w));
          const float alpha = m[nt][j] == -INFINITY ? 0.f : fast_exp2(m[nt][j] - t);
          m[nt][j] = t;
          l[nt][j] *= alpha;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            o[nt][k][j] *= alpha;
            o[nt][k][2 + j] *= alpha;
          }
        }
    }
    // ---- P^T, and O^T += V^T P^T
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], r1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float e0 = fast_exp2(s[kt][nt][2 * u] - r0), e1 = fast_exp2(s[kt][nt][2 * u + 1] - r1);
          l[nt][0] += e0;
          l[nt][1] += e1;
          pb[nt][u] = dec_transpose(BF ? pack_bf16x2(e0, e1) : pack_f16x2(e0, e1));
        }
      }
      const int r = kt * 16 + (KIND != DEC_E4M3 ? (lane & 7) + ((lane >> 4) & 1) * 8 : lane & 15);
      const uint32_t row_at = vs_base + r * C::ROW;
      const int x = swizzle(r);
      const int half = KIND != DEC_E4M3 ? (lane >> 3) & 1 : lane >> 4;
#pragma unroll
      for (int c = 0; c < C::CH / 2; ++c) {
        uint32_t f[4];
        dec_ldsm_t(row_at + (((2 * c + half) << 4) ^ x), f);
        if (KIND != DEC_E4M3) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) dec_mma<BF>(o[nt][c], f[0], f[1], f[2], f[3], pb[nt][0], pb[nt][1]);
        } else {
          // a register holds columns 2u, 2u + 1 of two keys: rows u and u + 8 of the fragment stand for these columns
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = __byte_perm(f[i], 0, 0x3120);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            dec_mma<false>(o[nt][2 * c % KSTEPS], dec_widen_e4m3(f[0]), dec_widen_e4m3(f[0] >> 16), dec_widen_e4m3(f[1]),
                           dec_widen_e4m3(f[1] >> 16), pb[nt][0], pb[nt][1]);
            dec_mma<false>(o[nt][(2 * c + 1) % KSTEPS], dec_widen_e4m3(f[2]), dec_widen_e4m3(f[2] >> 16),
                           dec_widen_e4m3(f[3]), dec_widen_e4m3(f[3] >> 16), pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (++cur.t < cur.nt && at + 1 < last) continue;

    // ---- end of a stretch or of the piece
    const int s0 = at + 1 - cur.t;  // where the stretch begins on the line
    const int b = cur.b, out_head = head0, out_heads = heads, out_kvh = kvh;
    const bool whole = cur.t == cur.nt && s0 >= first;
    const int done_hg = cur.hg, done_nt = cur.nt;
    if (at + 1 < last) {
      next_stretch(cur);
      load_q(cur);  // under what follows
    }
    fresh = true;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], w);
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float inv[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          inv[j] = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];
          if (KIND == DEC_E4M3) inv[j] *= a.v_scale[a.v_scale_n > 1 ? out_kvh : 0];
          const int h = nt * 8 + 2 * lane + j;
          if (a.lse && lane < 4 && h < out_heads)
            a.lse[(long long)b * a.heads + out_head + h] = m[nt][j] + log2f(l[nt][j]);
        }
        const int h = nt * 8 + lane / 4;  // after the transposition: heads are rows
        uint16_t* out = dec_out(p, b, out_head + h);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) {
          uint32_t x = dec_transpose(dec_pack_out(p, o[nt][k][0] * inv[0], o[nt][k][1] * inv[1]));
          uint32_t y = dec_transpose(dec_pack_out(p, o[nt][k][2] * inv[0], o[nt][k][3] * inv[1]));
          if (h < out_heads) {
            if (KIND != DEC_E4M3) {
              *reinterpret_cast<uint32_t*>(out + k * 16 + 2 * (lane & 3)) = x;
              *reinterpret_cast<uint32_t*>(out + k * 16 + 8 + 2 * (lane & 3)) = y;
            } else {
              *reinterpret_cast<uint2*>(out + k * 16 + 4 * (lane & 3)) =
                  make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
            }
          }
        }
      }
    } else {
      // part 2 w ends in this piece, part 2 w + 1 reaches its end
      const int part = 2 * warp + (at + 1 < last ? 0 : 1);
      if (lane == 0) parts[part] = DecPart{s0, b, done_hg, done_nt};
      float* dst = part_o(part);
      if (part & 1) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (lane < 4) part_ml[part * NH + nt * 8 + 2 * lane + j] = make_float2(m[nt][j], l[nt][j]);
          float* row = dst + (nt * 8 + 2 * (lane & 3) + j) * D;
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            if (KIND != DEC_E4M3) {
              row[k * 16 + lane / 4] = o[nt][k][j];
              row[k * 16 + 8 + lane / 4] = o[nt][k][2 + j];
            } else {
              *reinterpret_cast<float2*>(row + k * 16 + lane / 4 * 2) = make_float2(o[nt][k][j], o[nt][k][2 + j]);
            }
          }
        }
    }
  }

  // ---- merge the parts of this CTA, stretch by stretch (they lie in the order of the line), a warp per head
  __syncthreads();
  auto merge = [&](int i, int n, const DecPart& me, int turn) {  // parts i .. i + n - 1, without the empty ones
    const bool whole = me.s >= cta_first && me.s + me.nt <= cta_last;
    const int of_kv = me.hg / p.groups_per_kv, from = of_kv * p.group + (me.hg - of_kv * p.groups_per_kv) * NH;
    const int n_heads = min(NH, (of_kv + 1) * p.group - from);
    const long long row = ((long long)blockIdx.x * 2 + (me.s >= cta_first ? 1 : 0)) * NH;
    const float v_scale = KIND == DEC_E4M3 && whole ? a.v_scale[a.v_scale_n > 1 ? of_kv : 0] : 1.f;
    constexpr int HPW = D == 64 ? 2 : 1;  // heads at a time
    for (int h = (warp + turn) % DEC_WARPS * HPW + lane / (32 / HPW); h < n_heads; h += DEC_WARPS * HPW)
#pragma unroll
    for (int col = lane % (D / 4) * 4; col < D; col += 128) {
      float top = -INFINITY, sum = 0.f;
      for (int q = i; q < i + n; ++q)
        if (parts[q].s >= 0) top = fmaxf(top, part_ml[q * NH + h].x);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int q = i; q < i + n; ++q) {
        if (parts[q].s < 0) continue;
        const float2 ml = part_ml[q * NH + h];
        const float4 v = *reinterpret_cast<const float4*>(part_o(q) + h * D + col);
        const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
        sum += f * ml.y;
        x.x += f * v.x;
        x.y += f * v.y;
        x.z += f * v.z;
        x.w += f * v.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : v_scale / sum;
        *reinterpret_cast<uint2*>(dec_out(p, me.b, from + h) + col) =
            make_uint2(dec_pack_out(p, x.x * inv, x.y * inv), dec_pack_out(p, x.z * inv, x.w * inv));
        if (a.lse && col == 0) a.lse[(long long)me.b * a.heads + from + h] = top + log2f(sum);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (row + h) * D + col) = x;
        if (col == 0) p.part_ml[row + h] = make_float2(top, sum);
      }
    }
  };
  for (int i = 0, turn = 0; i < C::PARTS;) {
    const DecPart me = parts[i];
    int n = 1;
    if (me.s >= 0) {
      while (i + n < C::PARTS && (parts[i + n].s < 0 || parts[i + n].s == me.s)) ++n;
      merge(i, n, me, turn++);
    }
    i += n;
  }
}

// Joins the parts of the stretch that is cut at the start of CTA blockIdx.x's piece for the first time: the end of the
// CTA before, then the beginning of every CTA that it reaches into. One block per query head of the group; the first
// parts are loaded before their weights are known, for the kernel is a chain of loads and little else.
static constexpr int JOIN_THREADS = 128;
template <int D, int NH>
__global__ void __launch_bounds__(JOIN_THREADS) attention_decode_join_kernel(const __grid_constant__ DecodeParams p, int e4m3) {
  constexpr int COLS = D / 4, LANES = JOIN_THREADS / COLS;  // threads along a row, rows at a time
  constexpr int EARLY = 4, WARPS = JOIN_THREADS / 32;
  __shared__ float weight[1024];
  __shared__ float red[2][WARPS];
  __shared__ float4 acc[JOIN_THREADS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x, h = blockIdx.y;
  const DecMeta me = p.meta[c];
  const int per = *p.per;
  if (me.b < 0 || me.s >= per * c || me.s < per * (c - 1)) return;
  const int kvh = me.hg / p.groups_per_kv, head = kvh * p.group + me.hg % p.groups_per_kv * NH + h;
  if (head >= (kvh + 1) * p.group) return;
  const int parts = 1 + (me.e - 1) / per + 1 - c;  // at most the CTAs, which are at most 1024
  auto part_of = [&](int i) { return i == 0 ? ((long long)(c - 1) * 2 + 1) * NH + h : (long long)(c + i - 1) * 2 * NH + h; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = threadIdx.x % COLS, from = threadIdx.x / COLS;
  auto load = [&](int i) {
    return i < parts ? reinterpret_cast<const float4*>(p.part_o + part_of(i) * D)[col] : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float4 early[EARLY];
#pragma unroll
  for (int u = 0; u < EARLY; ++u) early[u] = load(from + u * LANES);
  float top = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += JOIN_THREADS) top = fmaxf(top, p.part_ml[part_of(i)].x);
#pragma unroll
  for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[0][w]);
  float sum = 0.f;
  for (int i = threadIdx.x; i < parts; i += JOIN_THREADS) {
    const float2 ml = p.part_ml[part_of(i)];
    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
    weight[i] = f;
    sum += f * ml.y;
  }
#pragma unroll
  for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += red[1][w];
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float f, const float4& v) {
    x.x += f * v.x;
    x.y += f * v.y;
    x.z += f * v.z;
    x.w += f * v.w;
  };
#pragma unroll
  for (int u = 0; u < EARLY; ++u)
    if (from + u * LANES < parts) add(weight[from + u * LANES], early[u]);
#pragma unroll 8
  for (int i = from + EARLY * LANES; i < parts; i += LANES) add(weight[i], load(i));
  acc[threadIdx.x] = x;
  __syncthreads();
  if (from == 0) {
    for (int i = 1; i < LANES; ++i) add(1.f, acc[i * COLS + col]);
    float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (e4m3) inv *= p.a.v_scale[p.a.v_scale_n > 1 ? kvh : 0];
    *reinterpret_cast<uint2*>(dec_out(p, me.b, head) + col * 4) =
        make_uint2(dec_pack_out(p, x.x * inv, x.y * inv), dec_pack_out(p, x.z * inv, x.w * inv));
    if (p.a.lse && col == 0) p.a.lse[(long long)me.b * p.a.heads + head] = top + log2f(sum);
  }
}

// What a call will launch: heads per group, CTAs, and the workspace they need.
struct DecPlan {
  int nh, ctas;
  size_t off_warp, off_ml, off_meta, off_per, bytes;
};
// A group of 8 query heads fills the narrow side of the mma; 16 per group halve the reads of K and V for larger groups
// (head dim 256 keeps 8: two accumulators of 256 columns do not fit the registers).
static int dec_heads(const tb200_attention_decode_args* a) { return a->heads / a->kv_heads > 8 && a->head_dim <= 128 ? 16 : 8; }
static DecPlan dec_plan(const tb200_attention_decode_args* a, int sms) {
  DecPlan d;
  d.nh = dec_heads(a);
  d.ctas = sms * (a->head_dim == 256 ? 1 : 2);
  const size_t parts = (size_t)d.ctas * 2 * d.nh;
  d.off_warp = parts * a->head_dim * sizeof(float);
  d.off_ml = d.off_warp + parts / 2 * DEC_WARPS * a->head_dim * sizeof(float);
  d.off_meta = d.off_ml + parts * sizeof(float2);
  d.off_per = d.off_meta + (size_t)d.ctas * sizeof(DecMeta);
  d.bytes = d.off_per + 16;
  return d;
}

template <int D, int KIND, int NT>
static int launch_decode(const DecodeParams& p, int ctas, cudaStream_t stream) {
  using C = DecCfg<D, KIND, NT>;
  static_assert(C::STAGES >= 3 && C::SMEM <= C::LIMIT, "shared memory budget");
  auto kfn = attention_decode_kernel<D, KIND, NT>;
  if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return TB200_ERR_CUDA;
  if (launch_overlapped(kfn, dim3((unsigned)ctas), DEC_WARPS * 32, C::SMEM, stream, p) != cudaSuccess) return TB200_ERR_CUDA;
  const dim3 join((unsigned)ctas, (unsigned)(p.group < C::NH ? p.group : C::NH));
  return cuda_err(
      launch_overlapped(attention_decode_join_kernel<D, C::NH>, join, JOIN_THREADS, 0, stream, p, (int)(KIND == DEC_E4M3)));
}

template <int D, int KIND>
static int launch_decode_heads(const DecodeParams& p, const DecPlan& plan, cudaStream_t stream) {
  if constexpr (D <= 128) {
    if (plan.nh == 16) return launch_decode<D, KIND, 2>(p, plan.ctas, stream);
  }
  return launch_decode<D, KIND, 1>(p, plan.ctas, stream);
}
template <int D>
static int launch_decode_kind(const DecodeParams& p, const DecPlan& plan, cudaStream_t stream) {
  return p.a.cache_dtype == TB200_E4M3  ? launch_decode_heads<D, DEC_E4M3>(p, plan, stream)
         : p.a.cache_dtype == TB200_F16 ? launch_decode_heads<D, DEC_F16>(p, plan, stream)
                                        : launch_decode_heads<D, DEC_BF16>(p, plan, stream);
}

static int dec_check(const tb200_attention_decode_args* a) {
  if (!a) return TB200_ERR_BAD_ARG;
  if (a->batch < 0 || a->heads < 0 || a->kv_heads < 1 || a->heads % a->kv_heads || a->n_pages < 0 || a->max_pages < 0 ||
      a->page_size < 1)
    return TB200_ERR_BAD_ARG;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return TB200_ERR_UNSUPPORTED;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  if (a->cache_dtype != TB200_E4M3 && a->cache_dtype != a->dtype) return TB200_ERR_UNSUPPORTED;
  if (a->batch > INT32_MAX || a->heads > (1 << 16) || a->batch * a->heads > INT32_MAX || a->max_pages > INT32_MAX ||
      a->n_pages > INT32_MAX ||
      a->max_pages * a->page_size > (1 << 30))
    return TB200_ERR_UNSUPPORTED;
  // The kernel's positions on the line of tiles are 32-bit, and the end of a CTA's piece is computed before it is cut to the
  // line's: up to 4 / 592 of the line behind it (4 warps a CTA, at least 148 CTAs), which 2^26 covers.
  const int64_t nh = dec_heads(a), hgs = (a->heads / a->kv_heads + nh - 1) / nh * a->kv_heads;
  const int64_t tiles = (a->max_pages * a->page_size + 15) / 16;  // of one sequence and head group, at most
  if (hgs * tiles > INT32_MAX || a->batch * (hgs * tiles) > INT32_MAX - (1 << 26)) return TB200_ERR_UNSUPPORTED;
  return TB200_OK;
}

}  // namespace tb200

using namespace tb200;

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

extern "C" size_t tb200_attention_decode_workspace_bytes(const tb200_attention_decode_args* a) {
  if (dec_check(a) != TB200_OK || a->batch == 0 || a->heads == 0) return 0;
  const int sms = sm_count();
  return sms > 0 ? dec_plan(a, sms).bytes : 0;
}

extern "C" int tb200_attention_decode(const tb200_attention_decode_args* a, void* stream_) {
  const int rc = dec_check(a);
  if (rc != TB200_OK) return rc;
  const bool c8 = a->cache_dtype == TB200_E4M3;
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
  if (a->batch == 0 || a->heads == 0) return TB200_OK;
  if (!a->q || !a->o || !a->seq_lens || (a->n_pages > 0 && (!a->k_cache || !a->v_cache)) ||
      (a->max_pages > 0 && !a->page_table) || (c8 && (!a->k_scale || !a->v_scale)))
    return TB200_ERR_BAD_ARG;
  const int sms = sm_count();
  if (sms <= 0) return TB200_ERR_CUDA;
  const DecPlan plan = dec_plan(a, sms);
  if (plan.ctas > 1024) return TB200_ERR_UNSUPPORTED;
  if (!a->workspace || off16(a->workspace) || a->workspace_bytes < plan.bytes) return TB200_ERR_BAD_ARG;
  DecodeParams p;
  memset(&p, 0, sizeof(p));
  p.a = *a;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.group = (int)(a->heads / a->kv_heads);
  p.groups_per_kv = (p.group + plan.nh - 1) / plan.nh;
  p.hgs = p.groups_per_kv * (int)a->kv_heads;
  p.max_len = (int)(a->max_pages * a->page_size);
  while ((1ll << p.page_shift) < a->page_size) ++p.page_shift;
  p.page_mul = (uint32_t)((1ull << (31 + p.page_shift)) / (uint64_t)a->page_size + 1);
  const int64_t size = c8 ? 1 : 2;
  p.k_page = a->kc_stride_page * size;
  p.k_tok = a->kc_stride_tok * size;
  p.k_head = a->kc_stride_head * size;
  p.v_page = a->vc_stride_page * size;
  p.v_tok = a->vc_stride_tok * size;
  p.v_head = a->vc_stride_head * size;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.warp_o = reinterpret_cast<float*>(ws + plan.off_warp);
  p.part_ml = reinterpret_cast<float2*>(ws + plan.off_ml);
  p.meta = reinterpret_cast<DecMeta*>(ws + plan.off_meta);
  p.per = reinterpret_cast<int*>(ws + plan.off_per);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return a->head_dim == 64 ? launch_decode_kind<64>(p, plan, stream)
         : a->head_dim == 128 ? launch_decode_kind<128>(p, plan, stream) : launch_decode_kind<256>(p, plan, stream);
}
