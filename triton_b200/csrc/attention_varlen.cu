// Flash-attention forward over packed sequences of different lengths, with grouped heads; keys and values packed too, or
// in the pages of a cache. O = softmax(Q K^T * sm_scale [+ causal mask]) V per sequence, base-2 log-sum-exp per row.
//
// The pipeline is that of attention.cu (warp 0 TMA loads, warp 1 issues every tcgen05.mma, two softmax warpgroups of 128
// query rows that alternate on the tensor pipe; S and P in tensor memory, O rescaled only when the running maximum grew
// by more than 2^8). What differs:
//   rows      A group's 128 rows are 128 / gp consecutive tokens x gp query heads of one kv head, gp a divisor of
//             heads / kv_heads: one box of a 4-D tensor map (column, head of the pack, token, pack). A tile so covers fewer
//             tokens, which wastes less on short sequences and on the causal diagonal, and K / V are read once per pack
//             instead of once per head.
//   schedule  attention_varlen_schedule_kernel turns the sequence offsets into a list of pieces, the longest KV walks
//             first; the lengths never pass through the host. The load warp of a CTA draws its next piece from a counter and
//             hands it to the other roles through shared memory.
//   split     A tile whose KV walk is longer than an even share of all work (few queries over a long cache, one sequence
//             among short ones) becomes several pieces: each leaves its accumulator, maxima and sums in the workspace, and
//             attention_varlen_join_kernel combines them in the order of the keys.
//   tails     The last KV block of a sequence runs into the next sequence's rows (or into whatever a page holds). Scores
//             there are replaced by -inf, so K's content is irrelevant; V's is not (0 * NaN), so warp 2 overwrites
//             those rows of the V tile with zeros in shared memory before the P V product may read it.
//   half      A tile whose tokens fit the first group (short sequences, ends) leaves the second group out.
//   pages     A KV block is 128 / r boxes of r = gcd(page size, 128) rows; the lanes of the load warp look up and issue one
//             page each. A page outside the pool is loaded from behind its end, which reads as zeros.
// Bound: the chain scores -> softmax -> P V of a group, 3400 cycles per 128 keys at D = 128 (of them 1790 softmax, 1024
// exponentials at the special-function unit's rate); tensor pipe about 60 %. Measured: 16001-token prompt, 32 / 8 heads of
// 128, 1226 TFLOP/s from cold, 1075 under the power limit; 24 prompts of 5 to 3000 tokens 240 us = 0.58 of the floor.
#include <limits.h>
#include <string.h>

#include "attention_common.cuh"
#include "common.cuh"
#include "host_common.h"

namespace tb200 {

static constexpr int VAR_THREADS = 384;
static constexpr int VAR_BN = 128;      // kv rows per block
static constexpr int VAR_MAX_STAGES = 4;
static constexpr float VAR_RESCALE_THRESHOLD = 8.0f;

// One piece of the schedule: n_tok tokens from packed row tok0 on over the KV blocks from j0 on; diag = the last key
// position that token 0 of the tile sees under a causal mask; n0 / n1 = KV blocks of the first / second group (n1 = 0: no
// tokens in it). part: this piece's slot in the workspace for the first pack, part_step slots further for each pack (part
// < 0: the tile is in one piece). In shared memory `part` is that of the pack, and n0 = 0 ends the list.
struct __align__(16) VarTile {
  int tok0, n_tok, kv_len, kv_first;
  int diag, n0, n1, j0;
  int part, part_step, pack, pad;
};
// A tile that was split: its parts lie at part + pack * n_parts + (0 .. n_parts - 1).
struct __align__(16) VarSplit {
  int tok0, n_tok, part, n_parts;
};
static constexpr int VAR_MIN_BLOCKS = 4;  // no piece is cut below this many KV blocks: starting one costs about two
// Longest walk: a producer that is done waits for the whole of it, and a wait ends after 2 s. 2^25 keys are 2^18 blocks of
// about 3400 cycles (128 x 2 queries, D = 128), 0.5 s at 1.9 GHz.
static constexpr int VAR_MAX_KEYS = 1 << 25;
struct VarCounters {
  int n_pieces, n_split, next, pad;
};

struct VarlenParams {
  CUtensorMap tmq;       // (D, gp, tokens, packs), box (64, gp, 128 / gp, 1), 128-byte swizzle
  CUtensorMap tmk, tmv;  // packed: (D, tokens, kv heads), box (64, 128, 1); pages: (D, page rows, kv heads, pages), box (64, r, 1, 1)
  void* o;
  float* lse;
  int* status;
  const VarTile* pieces;
  const VarSplit* splits;
  VarCounters* count;
  float* part_o;    // [part][rows of a tile][D]
  float2* part_ml;  // [part][rows of a tile]: maximum, sum
  const int32_t* page_table;
  long long table_stride, o_stride_tok, o_stride_head;
  int heads, packs, gp, packs_per_kv;
  int page_size, box_rows, n_pages, max_pages;
  int no_page;  // first page coordinate behind the pool: reads as zeros
  int causal;
  float scale_log2;
};

struct ScheduleParams {
  const int32_t *cu_q, *cu_k, *seq_lens;
  VarTile* pieces;
  VarSplit* splits;
  VarCounters* count;
  int batch, tokens_q, tokens_k, tile_tokens, group_tokens, causal, two_groups, paged;
  int max_len;  // pages: what the page table can hold
  int packs, ctas, max_pieces, max_splits, max_parts;
};

struct SeqExtent {
  int q0, q_len, k_len, k_first;
};
__device__ __forceinline__ SeqExtent seq_extent(const ScheduleParams& p, int b) {
  SeqExtent s;  // every offset is brought into its tensor before it is used: a wrong one costs results, not memory
  s.q0 = min(max(p.cu_q[b], 0), p.tokens_q);
  s.q_len = max(min(max(p.cu_q[b + 1], 0), p.tokens_q) - s.q0, 0);
  if (p.paged) {
    s.k_len = min(max(p.seq_lens[b], 0), p.max_len);
    s.k_first = b;
  } else {
    s.k_first = min(max(p.cu_k[b], 0), p.tokens_k);
    s.k_len = max(min(max(p.cu_k[b + 1], 0), p.tokens_k) - s.k_first, 0);
    if (s.k_len == 0) s.k_first = max(p.tokens_k, 1);  // behind the last row: the one block loaded for it is all zeros
  }
  return s;
}
__device__ __forceinline__ VarTile make_tile(const ScheduleParams& p, const SeqExtent& s, int i) {
  VarTile t;
  const int first = i * p.tile_tokens;
  t.tok0 = s.q0 + first;
  t.n_tok = min(s.q_len - first, p.tile_tokens);
  t.kv_len = s.k_len;
  t.kv_first = s.k_first;
  t.diag = first + s.k_len - s.q_len;
  auto blocks = [&](int tokens) {  // at least one: rows that see nothing still pass through the pipeline, fully masked
    const int seen = p.causal ? min(s.k_len, t.diag + tokens) : s.k_len;
    return max((seen + VAR_BN - 1) / VAR_BN, 1);
  };
  t.n0 = blocks(min(t.n_tok, p.group_tokens));
  t.n1 = p.two_groups && t.n_tok > p.group_tokens ? blocks(t.n_tok) : 0;
  t.j0 = 0;
  t.part = -1;
  t.part_step = t.pack = t.pad = 0;
  return t;
}

// One block. Cuts the tiles (below), then a counting sort of all pieces by their KV blocks, most first (a piece of one group
// takes as long as one of two: what counts is the longer walk; sorted by the sum, 5 unequal prompts over 32000 cached
// keys took 360 us instead of 290). One warp per sequence at a time. The order inside a bucket and the places of the parts
// are left to the atomics: they decide which CTA runs a piece and where its part lies, not what is computed.
//
// A tile of n blocks is cut into ceil(n / cap) even pieces with cap = all blocks of all packs / CTAs (at least
// VAR_MIN_BLOCKS): nothing is cut while every tile is shorter than an even share. Cut tiles number less than the CTAs and
// their pieces at most blocks / cap + cut tiles <= 2 CTAs, which bounds the workspace. 9 sequences of 62 queries over up to
// 20000 keys (24 / 8 heads of 256, 88 tiles): 548 us uncut, 190 us cut; finer pieces (cap / 2) gained nothing in a model of
// the schedule and double the parts. Takes 6 us, half of it under the end of the kernel before and the start of the next.
static constexpr int SCHED_BUCKETS = 1024;
__global__ void __launch_bounds__(1024) attention_varlen_schedule_kernel(const ScheduleParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ int count[SCHED_BUCKETS];
  __shared__ int warp_sum[32];
  __shared__ int n_split, n_parts;
  __shared__ unsigned long long all;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  count[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    all = 0;
    n_split = n_parts = 0;
  }
  __syncthreads();
  auto each_tile = [&](auto&& f) {
    for (int b = warp; b < p.batch; b += 32) {
      const SeqExtent s = seq_extent(p, b);
      const int n = (s.q_len + p.tile_tokens - 1) / p.tile_tokens;
      for (int i = lane; i < n; i += 32) f(make_tile(p, s, i));
    }
  };
  if (p.max_parts > 0) {
    unsigned long long mine = 0;
    each_tile([&](const VarTile& t) { mine += max(t.n0, t.n1); });
#pragma unroll
    for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0 && mine) atomicAdd(&all, mine);
    __syncthreads();
  }
  const unsigned long long work = all * p.packs;
  const int cap = max(work <= INT_MAX ? (int)work / p.ctas + 1 : (int)(work / p.ctas) + 1, VAR_MIN_BLOCKS);
  int shift = 0;  // a piece has at most cap + 1 blocks
  while (((cap + 1ll) >> shift) >= SCHED_BUCKETS) ++shift;
  auto bucket_of = [&](int blocks) { return SCHED_BUCKETS - 1 - min(blocks >> shift, SCHED_BUCKETS - 1); };
  // piece i of k even ones, the longer ones first; the last one also has the block that only the second group has
  auto cut = [](const VarTile& t, int i, int k) {
    if (k == 1) return t;
    VarTile x = t;
    const int even = t.n0 / k, more = t.n0 - even * k;
    x.j0 = i * even + min(i, more);
    const int end = x.j0 + even + (i < more ? 1 : 0);
    x.n0 = end - x.j0;
    if (t.n1 > 0) x.n1 = (i + 1 == k ? t.n1 : end) - x.j0;
    return x;
  };
  auto pieces_of = [&](const VarTile& t) { return t.n0 <= cap ? 1 : (t.n0 + cap - 1) / cap; };
  each_tile([&](const VarTile& t) {
    const int k = pieces_of(t);
    for (int i = 0; i < k; ++i) {
      const VarTile x = cut(t, i, k);
      atomicAdd(&count[bucket_of(max(x.n0, x.n1))], 1);
    }
  });
  __syncthreads();
  // exclusive prefix sum over the 1024 buckets (thread i owns bucket i)
  const int own = count[threadIdx.x];
  int sum = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += other;
  }
  if (lane == 31) warp_sum[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += other;
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  count[threadIdx.x] = sum - own + (warp ? warp_sum[warp - 1] : 0);
  __syncthreads();
  each_tile([&](const VarTile& t) {
    const int k = pieces_of(t);
    int part = -1;
    if (k > 1) {
      part = atomicAdd(&n_parts, k * p.packs);
      const int at = atomicAdd(&n_split, 1);
      // offsets that overlap (no sequence may) could need more: such a tile is left out
      if (part + k * p.packs > p.max_parts || at >= p.max_splits) part = -2;
      if (part >= 0) *reinterpret_cast<int4*>(p.splits + at) = make_int4(t.tok0, t.n_tok, part, k);
      else if (at < p.max_splits) *reinterpret_cast<int4*>(p.splits + at) = make_int4(t.tok0, 0, 0, k);
    }
    for (int i = 0; i < k; ++i) {
      const VarTile x = cut(t, i, k);
      const int at = atomicAdd(&count[bucket_of(max(x.n0, x.n1))], 1);
      if (at < p.max_pieces) {
        int4* dst = reinterpret_cast<int4*>(p.pieces + at);
        dst[0] = make_int4(x.tok0, part == -2 ? 0 : x.n_tok, x.kv_len, x.kv_first);
        dst[1] = make_int4(x.diag, x.n0, x.n1, x.j0);
        dst[2] = make_int4(part >= 0 ? part + i : -1, k, 0, 0);
      }
    }
  });
  __syncthreads();
  if (threadIdx.x == 0) {
    p.count->n_pieces = min(warp_sum[31], p.max_pieces);
    p.count->n_split = min(n_split, p.max_splits);
    p.count->next = p.ctas;  // a CTA's first piece is that of its own number
  }
}

// G = query groups per CTA: 2, or 1 for head dim 256 (tiles of 64 KB, an accumulator of 256 columns).
template <int D, int G>
struct VarSmem {
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int KV_STAGES = G == 2 ? VAR_MAX_STAGES : 2;
  static constexpr int Q_OFFSET = 0;
  static constexpr int KV_OFFSET = G * TILE_BYTES;
  static constexpr int BAR_OFFSET = KV_OFFSET + KV_STAGES * TILE_BYTES;
  static constexpr int NUM_BARS = 4 + 2 * VAR_MAX_STAGES + 16 + 4;
  static constexpr int TOTAL = BAR_OFFSET + NUM_BARS * 8 + 16 + 1024;
};

__device__ __forceinline__ void mbar_init_a(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
// mbar_wait with a 32-bit shared address, all of it inline: a call would cost the softmax warps registers
// (nap: nanoseconds of sleep between two looks, for a wait that is in no hurry)
__device__ __forceinline__ bool var_wait(uint32_t bar, uint32_t parity, int* status, int code, uint32_t nap = 0) {
  if (mbar_try_wait_a(bar, parity)) return true;
  uint64_t t0 = 0;
  uint32_t spins = 0;
  for (;;) {
    if (mbar_try_wait_a(bar, parity)) return true;
    if (nap) __nanosleep(nap);
    if (((++spins) & 0xff) == 0) {
      if (*reinterpret_cast<volatile int*>(status) != 0) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > TB200_WAIT_TIMEOUT_NS) {
        atomicCAS(status, 0, (code << 16) | (int)(blockIdx.x & 0xffff));
        return false;
      }
    }
  }
}
__device__ __forceinline__ void tma_load_3d_a(uint32_t dst, const CUtensorMap* tmap, uint32_t bar, int x, int y, int z,
                                              uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_a(uint32_t dst, const CUtensorMap* tmap, uint32_t bar, int c0, int c1, int c2,
                                            int c3, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "l"(policy)
      : "memory");
}

template <int D, bool F16, int G, bool PAGED>
__global__ void __launch_bounds__(VAR_THREADS, 1) attention_varlen_kernel(const __grid_constant__ VarlenParams p) {
  using L = VarSmem<D, G>;
  constexpr bool TWO = G == 2;
  constexpr uint32_t KV_STAGES = L::KV_STAGES;
  constexpr int DBOX = D / 64;
  constexpr int BOX_BYTES = 128 * 128;
  constexpr uint32_t S_COLS = 128;
  constexpr uint32_t O_COL0 = 2 * S_COLS;
  constexpr uint32_t TMEM_COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // barriers by their 32-bit shared address: one register for all of them
  const uint32_t smem_a = smem_u32(smem);
  const uint32_t bars = smem_a + L::BAR_OFFSET;
  const uint32_t q_full = bars;                                // [2]
  const uint32_t q_empty = bars + 2 * 8;                       // [2]
  const uint32_t kv_full = bars + 4 * 8;                       // [KV]
  const uint32_t kv_empty = kv_full + VAR_MAX_STAGES * 8;      // [KV]
  const uint32_t s_full = kv_empty + VAR_MAX_STAGES * 8;       // [2] MMA -> softmax: S_g ready
  const uint32_t p_full = s_full + 2 * 8;                      // [2][4] softmax -> MMA: 32-column chunk c of P_g written (128 arrivals)
  const uint32_t pv_done = p_full + 8 * 8;                     // [2] MMA -> softmax: last PV_g of the piece complete
  const uint32_t o_free = pv_done + 2 * 8;                     // [2] softmax -> MMA: O_g read out (128 arrivals)
  const uint32_t v_dirty = o_free + 2 * 8;                     // MMA -> warp 2: the V tile ahead holds rows behind the sequence's end
  const uint32_t v_clean = v_dirty + 8;                        // warp 2 -> MMA: those rows are zero
  const uint32_t t_full = v_clean + 8;                         // [2] loader -> others: piece r is in slot r % 2
  const uint32_t t_empty = t_full + 2 * 8;                     // [2] others -> loader: read (one arrival per warp that runs)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::BAR_OFFSET + (L::NUM_BARS) * 8);
  __shared__ VarTile tile_slot[2];  // a variable of its own, so that what is read from it is known to be warp-uniform

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tmq);
    tma_prefetch_desc(&p.tmk);
    tma_prefetch_desc(&p.tmv);
    for (int i = 0; i < 2; ++i) {
      mbar_init_a(q_full + 8 * (i), 1);
      mbar_init_a(q_empty + 8 * (i), 1);
      mbar_init_a(s_full + 8 * (i), 1);
      for (int c = 0; c < 4; ++c) mbar_init_a(p_full + 8 * (i * 4 + c), 128);
      mbar_init_a(pv_done + 8 * (i), 1);
      mbar_init_a(o_free + 8 * (i), 128);
    }
    for (int i = 0; i < VAR_MAX_STAGES; ++i) {
      mbar_init_a(kv_full + 8 * (i), 1);
      mbar_init_a(kv_empty + 8 * (i), 1);
    }
    mbar_init_a(v_dirty, 1);
    mbar_init_a(v_clean, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init_a(t_full + 8 * (i), 1);
      mbar_init_a(t_empty + 8 * (i), 2 + 4 * G);
    }
    mbar_init_fence();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the schedule
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  int* const status = p.status;
  const int group_tokens = 128 / p.gp;
  // The r-th piece of this CTA, for the one thread of a warp that asks.
  auto next_tile = [&](uint32_t r, VarTile& t, uint32_t nap) -> bool {
    if (!var_wait(t_full + 8 * (r & 1), (r >> 1) & 1, status, WAIT_ATTN, nap)) return false;
    const int4* src = reinterpret_cast<const int4*>(tile_slot + (r & 1));
    const int4 a = src[0], b = src[1], c = src[2];
    t = VarTile{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, 0};
    mbar_arrive_a(t_empty + 8 * (r & 1));
    return t.n0 > 0;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ loader (whole warp; lane 0 waits and counts)
    reg_dealloc<104>();
    const uint64_t pol_q = policy_evict_first();
    const uint64_t pol_kv = policy_evict_last();
    const int n_boxes = PAGED ? VAR_BN / p.box_rows : 1;
    const uint32_t q_bytes = (uint32_t)(group_tokens * p.gp) * (D * 2);
    const int units = p.count->n_pieces * p.packs;
    uint32_t pos = 0, tc0 = 0, tc1 = 0;
    bool ok = true;
    auto load_q = [&](int g, const VarTile& t, int pack) {
      if (lane == 0) {
        mbar_expect_tx_a(q_full + 8 * (g), q_bytes);
#pragma unroll
        for (int b = 0; b < DBOX; ++b)
          tma_load_4d_a(smem_a + L::Q_OFFSET + g * L::TILE_BYTES + b * BOX_BYTES, &p.tmq, q_full + 8 * g, b * 64, 0,
                      t.tok0 + g * group_tokens, pack, pol_q);
      }
    };
    // the page of this lane's box of KV block j
    auto page_of = [&](const VarTile& t, int j) -> int {
      if (!PAGED || lane >= n_boxes) return 0;
      const int at = (j * VAR_BN + lane * p.box_rows) / p.page_size;
      if (at >= p.max_pages) return p.no_page;
      const int page = p.page_table[t.kv_first * p.table_stride + at];
      return page >= 0 && page < p.n_pages ? page : p.no_page;
    };
    auto load_kv = [&](const CUtensorMap* tm, const VarTile& t, int kvh, int j, int page) -> bool {
      const uint32_t stage = pos % KV_STAGES;
      bool go = true;
      if (lane == 0) {
        go = var_wait(kv_empty + 8 * (stage), ((pos / KV_STAGES) & 1) ^ 1, status, WAIT_SMEM_EMPTY);
        if (go) mbar_expect_tx_a(kv_full + 8 * (stage), L::TILE_BYTES);
      }
      go = __shfl_sync(0xffffffffu, (int)go, 0) != 0;
      if (!go) return false;
      const uint32_t dst = smem_a + L::KV_OFFSET + stage * L::TILE_BYTES;
      if (PAGED) {
        if (lane < n_boxes) {
          const int in_page = (j * VAR_BN + lane * p.box_rows) % p.page_size;
#pragma unroll
          for (int b = 0; b < DBOX; ++b)
            tma_load_4d_a(dst + b * BOX_BYTES + lane * p.box_rows * 128, tm, kv_full + 8 * stage, b * 64, in_page, kvh, page,
                        pol_kv);
        }
      } else if (lane == 0) {
#pragma unroll
        for (int b = 0; b < DBOX; ++b)
          tma_load_3d_a(dst + b * BOX_BYTES, tm, kv_full + 8 * stage, b * 64, t.kv_first + j * VAR_BN, kvh, pol_kv);
      }
      ++pos;
      return true;
    };
    auto wait_q = [&](int g, uint32_t count) -> bool {
      bool go = true;
      if (lane == 0) go = var_wait(q_empty + 8 * (g), (count & 1) ^ 1, status, WAIT_SMEM_EMPTY);
      return __shfl_sync(0xffffffffu, (int)go, 0) != 0;
    };
    int unit = blockIdx.x;
    auto fetch = [&](int u) {
      VarTile t = {};  // n0 = 0: the end
      if (u < units) {
        const int4* src = reinterpret_cast<const int4*>(p.pieces + u / p.packs);
        const int4 a = src[0], b = src[1], c = src[2];
        const int pack = u % p.packs;
        t = VarTile{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x < 0 ? -1 : c.x + pack * c.y, c.y, pack, 0};
      }
      return t;
    };
    VarTile ahead = fetch(unit);
    for (uint32_t r = 0; ok; ++r) {
      const VarTile t = ahead;
      if (lane == 0) {
        ok = var_wait(t_empty + 8 * (r & 1), ((r >> 1) & 1) ^ 1, status, WAIT_ATTN);
        if (ok) {
          tile_slot[r & 1] = t;
          mbar_arrive_a(t_full + 8 * (r & 1));
        }
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      if (!ok || t.n0 == 0) break;
      const int kvh = t.pack / p.packs_per_kv;
      const int n = max(t.n0, t.n1), end = t.j0 + n;
      // The next piece is drawn two blocks ahead of this one's end and looked up a block later: any later and the ring
      // would run empty, much earlier (all second pieces at once, in whatever order the CTAs start) cost a quarter on
      // two unequal pieces per CTA.
      int next = 0;
      auto draw = [&](int j) {
        if (j == max(end - 2, t.j0) && lane == 0) next = atomicAdd(&p.count->next, 1);
        if (j == end - 1) ahead = fetch(__shfl_sync(0xffffffffu, next, 0));
      };
      int page = page_of(t, t.j0), page_ahead = n > 1 ? page_of(t, t.j0 + 1) : 0;
      if (!wait_q(0, tc0++)) break;
      load_q(0, t, t.pack);
      if (!load_kv(&p.tmk, t, kvh, t.j0, page)) break;
      if (TWO && t.n1 > 0) {
        if (!wait_q(1, tc1++)) break;
        load_q(1, t, t.pack);
      }
      if (!load_kv(&p.tmv, t, kvh, t.j0, page)) break;
      draw(t.j0);
      for (int j = t.j0 + 1; j < end && ok; ++j) {
        page = page_ahead;
        if (j + 1 < end) page_ahead = page_of(t, j + 1);
        draw(j);
        ok = load_kv(&p.tmk, t, kvh, j, page) && load_kv(&p.tmv, t, kvh, j, page);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    reg_dealloc<104>();
    if (lane == 0) {
      const uint32_t idesc_qk = make_idesc(1u, 1u, 0u, 0u, 128, VAR_BN);   // bf16 x bf16, both K-major
      const uint32_t idesc_pv = make_idesc(1u, 1u, 0u, 1u, 128, D);        // B (= V) MN-major
      constexpr uint32_t fmt_fix = F16 ? ((1u << 7) | (1u << 10)) : 0u;   // fp16: operand format 0
      const uint32_t idq = idesc_qk & ~fmt_fix, idp = idesc_pv & ~fmt_fix;
      const uint64_t qdesc0 = make_smem_desc(smem_a + L::Q_OFFSET, 16, 1024, SWIZZLE_128B);
      const uint64_t kdesc0 = make_smem_desc(smem_a + L::KV_OFFSET, 16, 1024, SWIZZLE_128B);
      const uint64_t vdesc0 = make_smem_desc(smem_a + L::KV_OFFSET, BOX_BYTES, 1024, SWIZZLE_128B);
      uint32_t kvs = 0, kvph = 0;           // ring position of the next unconsumed KV tile
      uint32_t it0 = 0, it1 = 0;            // KV blocks issued so far per group (phases of the s / p barriers)
      uint32_t tc0 = 0, tc1 = 0, clean = 0; // tiles per group, cleaned V tiles
      bool ok = true;

      auto issue_qk = [&](int g, uint32_t kstage) {
        const uint64_t qd = qdesc0 + (uint64_t)((g * L::TILE_BYTES) >> 4);
        const uint64_t kd = kdesc0 + (uint64_t)((kstage * L::TILE_BYTES) >> 4);
        const uint32_t d_s = tmem_base + g * S_COLS;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t off = (uint64_t)(((k >> 2) * BOX_BYTES + (k & 3) * 32) >> 4);
          umma_f16_ss(d_s, qd + off, kd + off, idq, k > 0 ? 1u : 0u);
        }
        umma_commit_a(s_full + 8 * (g));
      };
      // PV_g at once when all of P_g is there (`ready`: its last chunk was seen; a thread arrives on the chunk barriers in
      // order), else in four slices of 32 keys, each as soon as the softmax has published that chunk. In steady state the
      // tensor pipe is the slower side and P_g waits for it: the waits and fences between slices of two MMAs then only
      // left it idle.
      auto issue_pv = [&](int g, uint32_t vstage, uint32_t accum, uint32_t iph, bool ready, bool last) -> bool {
        const uint64_t vd = vdesc0 + (uint64_t)((vstage * L::TILE_BYTES) >> 4);
        const uint32_t d_o = tmem_base + O_COL0 + g * D;
        const uint32_t a_p = tmem_base + g * S_COLS;
        if (ready) {
          tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ts(d_o, a_p + k * 8, vd + (uint64_t)((k * 16 * 128) >> 4), idp, (k > 0) ? 1u : accum);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (!var_wait(p_full + 8 * (g * 4 + c), iph, status, WAIT_ATTN)) return false;
            tc_fence_after_sync();
#pragma unroll
            for (int k = 2 * c; k < 2 * (c + 1); ++k)
              umma_f16_ts(d_o, a_p + k * 8, vd + (uint64_t)((k * 16 * 128) >> 4), idp, (k > 0) ? 1u : accum);
          }
        }
        if (last) umma_commit_a(pv_done + 8 * (g));
        return true;
      };
      auto advance = [&]() {
        if (++kvs == KV_STAGES) {
          kvs = 0;
          kvph ^= 1;
        }
      };

      // One stream of blocks across the pieces: the first scores of the next piece are issued where the next block's would
      // be, between the last P V of the two groups, so they are there when a group has written its results out.
      uint32_t r = 0;
      VarTile t, u;
      bool have = next_tile(r, t, 0);
      u = t;
      for (bool first = true; have;) {
        const int n0 = t.n0, n1 = TWO ? t.n1 : 0, n = max(n0, n1);
        const bool both = TWO && n1 > 0;
        const uint32_t tph0 = tc0++ & 1, tph1 = tc1 & 1;
        if (both) ++tc1;
        // A walk that ends behind the sequence's end: its last V tile is cleaned before use. The helper is told once the
        // full phase before that tile's in its ring stage has been seen here, so its wait cannot mistake an earlier phase
        // for it, and not again before it has answered.
        const bool tail = (t.j0 + n) * VAR_BN > t.kv_len;
        // S_g(0) = Q_g K(0)^T of piece x (its K tile in stage k): called for each group in its place
        auto begin0 = [&](const VarTile& x, uint32_t k, uint32_t qph) -> bool {
          if (!var_wait(q_full, qph, status, WAIT_ATTN)) return false;
          tc_fence_after_sync();
          issue_qk(0, k);
          if (x.n0 == 1) umma_commit_a(q_empty);
          return true;
        };
        auto begin1 = [&](const VarTile& x, uint32_t k, uint32_t qph) -> bool {
          if (TWO && x.n1 > 0) {
            if (!var_wait(q_full + 8, qph, status, WAIT_ATTN)) return false;
            tc_fence_after_sync();
            issue_qk(1, k);
          }
          umma_commit_a(kv_empty + 8 * k);
          if (TWO && x.n1 == 1) umma_commit_a(q_empty + 8);
          const int blocks = max(x.n0, TWO ? x.n1 : 0);
          if (blocks == 1 && (x.j0 + 1) * VAR_BN > x.kv_len) mbar_arrive_a(v_dirty);
          return true;
        };
        if (first) {
          first = false;
          const uint32_t k = kvs, kph = kvph;
          advance();
          if (!var_wait(kv_full + 8 * k, kph, status, WAIT_SMEM_FULL) || !begin0(t, k, tph0) || !begin1(t, k, tph1)) break;
        }
        // the second group's diagonal lies at most 128 keys behind the first one's: n0 is n1 or n1 - 1
        // All blocks but the last: this loop is kept free of everything that only borders of pieces need. What its thread
        // does between two tcgen05.mma is idle time of the tensor pipe.
        for (int j = 0; j + 1 < n; ++j) {
          const uint32_t iph0 = it0++ & 1, iph1 = it1 & 1;
          const bool more0 = j + 1 < n0;
          const uint32_t vcur = kvs, vcur_ph = kvph;
          advance();
          const uint32_t knext = kvs, knext_ph = kvph;
          advance();
          if (!var_wait(kv_full + 8 * vcur, vcur_ph, status, WAIT_SMEM_FULL)) { ok = false; break; }
          if (tail && j == n - 2) mbar_arrive_a(v_dirty);
          const bool k_ready = mbar_test_a(kv_full + 8 * knext, knext_ph);
          if (j == 0 && !var_wait(o_free, tph0 ^ 1, status, WAIT_ATTN)) { ok = false; break; }
          if (!issue_pv(0, vcur, j > 0 ? 1u : 0u, iph0, mbar_test_a(p_full + 8 * 3, iph0), !more0)) { ok = false; break; }
          if (!k_ready && !var_wait(kv_full + 8 * knext, knext_ph, status, WAIT_SMEM_FULL)) { ok = false; break; }
          tc_fence_after_sync();
          if (more0) {
            issue_qk(0, knext);
            if (j + 2 == n0) umma_commit_a(q_empty);
          }
          const bool p1_ready = both && mbar_test_a(p_full + 8 * 7, iph1);
          if (both) {
            if (j == 0 && !var_wait(o_free + 8, tph1 ^ 1, status, WAIT_ATTN)) { ok = false; break; }
            if (!issue_pv(1, vcur, j > 0 ? 1u : 0u, iph1, p1_ready, false)) { ok = false; break; }
            ++it1;
          }
          umma_commit_a(kv_empty + 8 * vcur);
          if (both) issue_qk(1, knext);
          umma_commit_a(kv_empty + 8 * knext);
          if (both && j + 2 == n1) umma_commit_a(q_empty + 8);
        }
        if (!ok) break;
        // the last block, with the first scores of the next piece
        const uint32_t accum = n > 1 ? 1u : 0u;
        const uint32_t vcur = kvs, vcur_ph = kvph;
        advance();
        if (!var_wait(kv_full + 8 * vcur, vcur_ph, status, WAIT_SMEM_FULL)) break;
        if (tail) {
          if (!var_wait(v_clean, clean++ & 1, status, WAIT_ATTN)) break;
          tc_fence_after_sync();
        }
        if (n0 == n) {
          if (n == 1 && !var_wait(o_free, tph0 ^ 1, status, WAIT_ATTN)) break;
          if (!issue_pv(0, vcur, accum, it0++ & 1, false, true)) break;
        }
        have = next_tile(++r, u, 0);
        uint32_t knext = 0;
        if (have) {
          knext = kvs;
          const uint32_t knext_ph = kvph;
          advance();
          if (!var_wait(kv_full + 8 * knext, knext_ph, status, WAIT_SMEM_FULL)) break;
          if (!begin0(u, knext, tc0 & 1)) break;
        }
        if (both) {
          if (n == 1 && !var_wait(o_free + 8, tph1 ^ 1, status, WAIT_ATTN)) break;
          if (!issue_pv(1, vcur, accum, it1++ & 1, false, true)) break;
        }
        umma_commit_a(kv_empty + 8 * vcur);
        if (have && !begin1(u, knext, tc1 & 1)) break;
        t = u;
      }
    }
  } else if (warp == 3) {
    reg_dealloc<104>();  // only takes part in the warpgroup-wide register release
  } else if (warp == 2) {
    // ------------------------------------------------------------------ V rows behind the end of a sequence
    reg_dealloc<104>();
    uint32_t pos = 0, told = 0;
    for (uint32_t r = 0;; ++r) {
      // Waits here nap and one lane has them: polled at full rate by two warps they took a tenth from the softmax warps.
      // The MMA warp says v_dirty a whole block ahead of its need.
      int stage = -1, first = 0;
      if (lane == 0) {
        VarTile t;
        if (next_tile(r, t, 32)) {
          const int n = max(t.n0, t.n1);
          const uint32_t at = pos + 2 * (n - 1) + 1;
          pos += 2 * n;
          stage = KV_STAGES;  // nothing to clean
          if ((t.j0 + n) * VAR_BN > t.kv_len) {  // only the last block of a walk can reach behind the end
            stage = at % KV_STAGES;
            first = max(t.kv_len - (t.j0 + n - 1) * VAR_BN, 0);  // row r of a box lies in its bytes [128 r, 128 r + 128)
            if (!var_wait(v_dirty, told++ & 1, status, WAIT_ATTN, 32) ||
                !var_wait(kv_full + 8 * stage, (at / KV_STAGES) & 1, status, WAIT_SMEM_FULL, 20))
              stage = -1;
          }
        }
      }
      stage = __shfl_sync(0xffffffffu, stage, 0);
      first = __shfl_sync(0xffffffffu, first, 0);
      if (stage < 0) break;
      if (stage < (int)KV_STAGES) {
        uint8_t* rows = smem + L::KV_OFFSET + stage * L::TILE_BYTES;
        for (int at = first * 128 + lane * 16; at < BOX_BYTES; at += 512)
#pragma unroll
          for (int box = 0; box < DBOX; ++box) *reinterpret_cast<uint4*>(rows + box * BOX_BYTES + at) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_a(v_clean);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax / correction / epilogue
    reg_alloc<192>();
    const int g = (warp - 4) >> 2;
    const int q = warp & 3;
    const int row = q * 32 + lane;                       // row of the group
    // token of the tile (behind every tile where the 128 rows are not whole tokens) and head of the pack, in one register:
    // 128 scores and little else fit the loop below
    const int place = (row < group_tokens * p.gp ? g * group_tokens + row / p.gp : 0x4000) | (row % p.gp) << 16;
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t t_s = tmem_base + lane_off + g * S_COLS;
    const uint32_t t_o = tmem_base + lane_off + O_COL0 + g * D;
    const float scale = p.scale_log2;
    uint32_t it = 0, tcount = 0;
    bool ok = true;
    for (uint32_t r = 0; ok && (TWO || g == 0); ++r) {
      // what the loop needs of the piece; the rest is read again behind it, so the slot is given back only there
      if (!var_wait(t_full + 8 * (r & 1), (r >> 1) & 1, status, WAIT_ATTN)) break;
      const volatile VarTile* slot = tile_slot + (r & 1);
      if (slot->n0 == 0) break;
      const int n = g == 0 ? slot->n0 : slot->n1;
      auto give_back = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive_a(t_empty + 8 * (r & 1));
      };
      if (n == 0) {
        give_back();
        continue;
      }
      float m = -INFINITY, l = 0.f;
      const int kv_last = slot->kv_len - 1, diag = slot->diag;
      // this row's last visible key, and that of the group's first row, counted from the block in hand
      int last = (p.causal ? min(kv_last, diag + (place & 0xffff)) : kv_last) - slot->j0 * VAR_BN;
      int safe = (p.causal ? min(kv_last, diag + g * group_tokens) : kv_last) - slot->j0 * VAR_BN;
      for (int j = 0; j < n; ++j, ++it, last -= VAR_BN, safe -= VAR_BN) {
        if (!var_wait(s_full + 8 * (g), it & 1, status, WAIT_ATTN)) { ok = false; break; }
        tc_fence_after_sync();
        uint32_t sv[128];
        tmem_ld_row32<0>(t_s, sv);
        tmem_ld_row32<32>(t_s + 32, sv);
        tmem_ld_row32<64>(t_s + 64, sv);
        tmem_ld_row32<96>(t_s + 96, sv);
        tmem_ld_wait();
        if (VAR_BN - 1 > safe) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i > last) sv[i] = 0xff800000u;  // -inf: contributes exp2(-inf) = 0
        }
        float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 128; i += 4) {
          mx0 = fmaxf(mx0, __uint_as_float(sv[i]));
          mx1 = fmaxf(mx1, __uint_as_float(sv[i + 1]));
          mx2 = fmaxf(mx2, __uint_as_float(sv[i + 2]));
          mx3 = fmaxf(mx3, __uint_as_float(sv[i + 3]));
        }
        const float m_blk = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * scale;  // scale > 0
        float alpha = 1.f;
        if (j == 0) {
          m = m_blk;
        } else if (m_blk - m > VAR_RESCALE_THRESHOLD) {
          alpha = fast_exp2(m - m_blk);
          m = m_blk;
        }
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // PV_g(j-1) is complete: it precedes S_g(j) in the MMA stream, and S_g(j) has arrived
          l *= alpha;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(t_o + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
            tmem_st_32x32b_x32(t_o + c, v);
          }
          tmem_st_wait();
        }
        // P = exp2(S * scale - m); a row that has seen nothing yet keeps its zeros (-inf - 0)
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t scale2 = pack2(scale, scale);
        const uint64_t negm2 = pack2(-ref, -ref);
        uint64_t sum2 = pack2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t x = fma2(pack2(__uint_as_float(sv[c + i]), __uint_as_float(sv[c + i + 1])), scale2, negm2);
            float x0, x1;
            unpack2(x, x0, x1);
            const float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
            sum2 = add2(sum2, pack2(e0, e1));
            pk[i >> 1] = F16 ? pack_f16x2(e0, e1) : pack_bf16x2(e0, e1);
          }
          if (c > 0) {
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive_a(p_full + 8 * (g * 4 + (c >> 5) - 1));
          }
          tmem_st_32x32b_x16(t_s + (c >> 1), pk);
        }
        float sum_lo, sum_hi;
        unpack2(sum2, sum_lo, sum_hi);
        l += sum_lo + sum_hi;
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive_a(p_full + 8 * (g * 4 + 3));
      }
      if (!ok) break;
      if (!var_wait(pv_done + 8 * (g), tcount++ & 1, status, WAIT_ATTN)) break;
      tc_fence_after_sync();
      const int tok_row = place & 0xffff;
      const bool valid = tok_row < slot->n_tok;
      const long long token = slot->tok0 + tok_row;
      const int head = slot->pack * p.gp + (place >> 16), part = slot->part;
      give_back();
      if (part >= 0) {
        // a piece of a split tile: the accumulator as it is
        const long long at = (long long)part * (G * 128) + g * 128 + row;
        float* dst = p.part_o + at * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_o + c, v);
          tmem_ld_wait();
          if (c + 32 == D) {
            tc_fence_before_sync();
            mbar_arrive_a(o_free + 8 * (g));
          }
          if (valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c + 8 * i), "r"(v[8 * i]),
                           "r"(v[8 * i + 1]), "r"(v[8 * i + 2]), "r"(v[8 * i + 3]), "r"(v[8 * i + 4]), "r"(v[8 * i + 5]),
                           "r"(v[8 * i + 6]), "r"(v[8 * i + 7])
                           : "memory");
          }
        }
        if (valid) p.part_ml[at] = make_float2(m, l);
        continue;
      }
      const float inv_l = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no visible key: zeros; NaN stays NaN
      uint16_t* orow = reinterpret_cast<uint16_t*>(p.o) + token * p.o_stride_tok + head * p.o_stride_head;
      const bool wide_st = (reinterpret_cast<uintptr_t>(orow) & 31) == 0;
      auto store32 = [&](const uint32_t (&v)[32], int c) {
        if (!valid) return;
        uint32_t w[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const float lo = __uint_as_float(v[2 * u]) * inv_l;
          const float hi = __uint_as_float(v[2 * u + 1]) * inv_l;
          w[u] = F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
        }
        if (wide_st) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(orow + c + 16 * i), "r"(w[8 * i]),
                         "r"(w[8 * i + 1]), "r"(w[8 * i + 2]), "r"(w[8 * i + 3]), "r"(w[8 * i + 4]), "r"(w[8 * i + 5]),
                         "r"(w[8 * i + 6]), "r"(w[8 * i + 7])
                         : "memory");
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            reinterpret_cast<uint4*>(orow + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
      };
      {
        uint32_t v0[32], v1[32];
        tmem_ld_32x32b_x32(t_o, v0);
#pragma unroll 1
        for (int c = 0; c < D; c += 64) {
          tmem_ld_wait();
          tmem_ld_32x32b_x32(t_o + c + 32, v1);
          store32(v0, c);
          tmem_ld_wait();
          if (c + 64 < D) {
            tmem_ld_32x32b_x32(t_o + c + 64, v0);
          } else {
            tc_fence_before_sync();
            mbar_arrive_a(o_free + 8 * (g));
          }
          store32(v1, c + 32);
        }
      }
      if (valid && p.lse) p.lse[token * p.heads + head] = m + log2f(l);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Combines the parts of split tiles: a warp per row, block (x, y) = rows 32 y .. of the x-th (split tile, pack).
template <int D, int G, bool F16>
__global__ void __launch_bounds__(256) attention_varlen_join_kernel(const __grid_constant__ VarlenParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x >= p.count->n_split * p.packs) return;
  const int4 e = *reinterpret_cast<const int4*>(p.splits + blockIdx.x / p.packs);
  const VarSplit s{e.x, e.y, e.z, e.w};
  const int pack = blockIdx.x % p.packs, group_tokens = 128 / p.gp;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = blockIdx.y * 32 + warp; r < (int)blockIdx.y * 32 + 32; r += 8) {
    const int row = r & 127, tok_row = (r >> 7) * group_tokens + row / p.gp;
    if (row >= group_tokens * p.gp || tok_row >= s.n_tok) continue;
    constexpr int ROWS = G * 128;
    const long long first = (long long)(s.part + pack * s.n_parts) * ROWS + r;
    float top = -INFINITY;
    for (int i = lane; i < s.n_parts; i += 32) top = fmaxf(top, p.part_ml[first + i * ROWS].x);
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    constexpr int COLS = D / 32;
    float x[COLS] = {}, sum = 0.f;
#pragma unroll 4
    for (int i = 0; i < s.n_parts; ++i) {
      const float2 ml = p.part_ml[first + i * ROWS];
      const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
      sum += f * ml.y;
      const float* src = p.part_o + (first + i * ROWS) * D + lane * COLS;
#pragma unroll
      for (int c = 0; c < COLS; c += 2) {
        const float2 v = *reinterpret_cast<const float2*>(src + c);
        x[c] += f * v.x;
        x[c + 1] += f * v.y;
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
    const long long token = s.tok0 + tok_row;
    const int head = pack * p.gp + row % p.gp;
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.o) + token * p.o_stride_tok + head * p.o_stride_head + lane * COLS;
#pragma unroll
    for (int c = 0; c < COLS; c += 2)
      *reinterpret_cast<uint32_t*>(dst + c) =
          F16 ? pack_f16x2(x[c] * inv, x[c + 1] * inv) : pack_bf16x2(x[c] * inv, x[c + 1] * inv);
    if (p.lse && lane == 0) p.lse[token * p.heads + head] = top + log2f(sum);
  }
}

template <int D, int G, bool PAGED>
static int launch_varlen(const VarlenParams& p, bool f16, int grid, int max_split, cudaStream_t stream) {
  using L = VarSmem<D, G>;
  static_assert(L::TOTAL + 2 * sizeof(VarTile) <= 232448, "shared memory budget");
  auto kfn = f16 ? attention_varlen_kernel<D, true, G, PAGED> : attention_varlen_kernel<D, false, G, PAGED>;
  if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL) != cudaSuccess)
    return TB200_ERR_CUDA;
  // starts while the schedule is being made: barriers and tensor memory are set up by the time it is there
  if (launch_overlapped(kfn, dim3((unsigned)grid), VAR_THREADS, L::TOTAL, stream, p) != cudaSuccess) return TB200_ERR_CUDA;
  if (max_split == 0) return TB200_OK;
  return cuda_err(launch_overlapped(f16 ? attention_varlen_join_kernel<D, G, true> : attention_varlen_join_kernel<D, G, false>,
                                    dim3((unsigned)max_split, 4 * G), 256, 0, stream, p));
}

struct VarPlan {
  int gp, packs, tile_tokens, group_tokens, ctas, max_split, max_parts;
  int64_t max_pieces;
  size_t off_splits, off_ml, off_o, bytes;
};
// gp: the largest divisor of the group that leaves at most 8 of a group's 128 rows unused (1 always does).
static VarPlan var_plan(const tb200_attention_varlen_args* a) {
  const int found = sm_count(), sms = found > 0 ? found : 148;  // a size can be asked for without a device
  VarPlan v;
  const int64_t group = a->heads / a->kv_heads;
  v.gp = (int)(group < 128 ? (group > 0 ? group : 1) : 128);
  while (group % v.gp || 128 / v.gp * v.gp < 120) --v.gp;
  v.packs = (int)(a->heads / v.gp);
  v.group_tokens = 128 / v.gp;
  v.tile_tokens = (a->head_dim == 256 ? 1 : 2) * v.group_tokens;
  const int64_t tiles = a->tokens_q / v.tile_tokens + a->batch;  // every sequence ends in at most one tile that is not full
  // walks of at most VAR_MIN_BLOCKS blocks are never cut
  const int64_t most_keys = a->page_size > 0 ? a->max_pages * a->page_size : a->tokens_k;
  const bool cuts = most_keys > (int64_t)VAR_MIN_BLOCKS * VAR_BN;
  v.max_split = cuts ? sms : 0;
  v.max_parts = cuts ? 2 * sms : 0;
  v.max_pieces = tiles + v.max_parts;
  const int64_t units = v.max_pieces * v.packs;
  v.ctas = (int)(units < sms ? (units > 0 ? units : 1) : sms);
  v.off_splits = 32 + (size_t)v.max_pieces * sizeof(VarTile);
  v.off_ml = (v.off_splits + (size_t)v.max_split * sizeof(VarSplit) + 31) / 32 * 32;
  const size_t part_rows = (size_t)v.max_parts * (a->head_dim == 256 ? 128 : 256);
  v.off_o = v.off_ml + part_rows * sizeof(float2);
  v.bytes = v.off_o + part_rows * a->head_dim * sizeof(float);
  return v;
}
static bool var_sizes_ok(const tb200_attention_varlen_args* a) {
  return a && a->batch >= 0 && a->heads >= 0 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 && a->tokens_q >= 0 &&
         a->tokens_k >= 0 && a->page_size >= 0 && a->n_pages >= 0 && a->max_pages >= 0;
}

}  // namespace tb200

using namespace tb200;

extern "C" size_t tb200_attention_varlen_workspace_bytes(const tb200_attention_varlen_args* a) {
  if (!var_sizes_ok(a)) return 0;
  return var_plan(a).bytes;
}

extern "C" int tb200_attention_varlen_fwd(const tb200_attention_varlen_args* a, void* stream_) {
  if (!var_sizes_ok(a)) return TB200_ERR_BAD_ARG;
  const bool paged = a->page_size > 0;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return TB200_ERR_UNSUPPORTED;
  if (a->dtype != TB200_BF16 && a->dtype != TB200_F16) return TB200_ERR_UNSUPPORTED;
  if (paged && a->page_size % 8) return TB200_ERR_UNSUPPORTED;
  if (!(a->sm_scale > 0.f)) return TB200_ERR_BAD_ARG;
  const int64_t strides[] = {a->q_stride_tok, a->q_stride_head, a->o_stride_tok, a->o_stride_head, a->k_stride_tok,
                             a->k_stride_head, a->v_stride_tok, a->v_stride_head,
                             paged ? a->k_stride_page : a->k_stride_tok, paged ? a->v_stride_page : a->v_stride_tok};
  for (int64_t s : strides)
    if (s % 8 || s < a->head_dim) return TB200_ERR_BAD_ARG;
  if (a->tokens_q > (1 << 30) || a->tokens_k > VAR_MAX_KEYS || a->batch > (1 << 30) || a->heads > (1 << 16) ||
      a->n_pages > (1 << 30) || (paged && (a->max_pages > VAR_MAX_KEYS || a->max_pages * a->page_size > VAR_MAX_KEYS)))
    return TB200_ERR_UNSUPPORTED;
  if (a->tokens_q == 0 || a->batch == 0 || a->heads == 0) return TB200_OK;
  if (!a->q || !a->o || !a->cu_seqlens_q) return TB200_ERR_BAD_ARG;
  if (paged ? ((!a->page_table && a->max_pages > 0) || !a->seq_lens) : !a->cu_seqlens_k) return TB200_ERR_BAD_ARG;
  // a pool or a packed tensor without rows has no address: the tensor maps are laid over q, no coordinate lies in them
  const bool keys = paged ? a->n_pages > 0 : a->tokens_k > 0;
  if (keys && (!a->k || !a->v)) return TB200_ERR_BAD_ARG;
  const void* bases[] = {a->q, keys ? a->k : a->q, keys ? a->v : a->q, a->o};
  for (const void* b : bases)
    if (reinterpret_cast<uintptr_t>(b) & 15) return TB200_ERR_BAD_ARG;
  const VarPlan plan = var_plan(a);
  if (plan.max_pieces * plan.packs > INT32_MAX / 2) return TB200_ERR_UNSUPPORTED;
  if (!a->workspace || a->workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(a->workspace) & 31))
    return TB200_ERR_BAD_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);

  VarlenParams p;
  memset(&p, 0, sizeof(p));
  const int D = a->head_dim;
  const bool f16 = a->dtype == TB200_F16;
  const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  {
    const uint64_t gp = plan.gp;
    const uint64_t dims[4] = {(uint64_t)D, gp, (uint64_t)a->tokens_q, (uint64_t)plan.packs};
    const uint64_t str[3] = {(uint64_t)a->q_stride_head * 2, (uint64_t)a->q_stride_tok * 2, gp * a->q_stride_head * 2};
    const uint32_t box[4] = {64, (uint32_t)gp, (uint32_t)plan.group_tokens, 1};
    const int rc = encode_tmap(&p.tmq, dt, 4, a->q, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != TB200_OK) return rc;
  }
  int box_rows = VAR_BN;
  for (int i = 0; i < 2; ++i) {
    const void* base = bases[1 + i];
    CUtensorMap* tm = i ? &p.tmv : &p.tmk;
    const int64_t st = i ? a->v_stride_tok : a->k_stride_tok, sh = i ? a->v_stride_head : a->k_stride_head;
    int rc;
    if (paged) {
      while (a->page_size % box_rows) box_rows >>= 1;
      const uint64_t dims[4] = {(uint64_t)D, (uint64_t)a->page_size, (uint64_t)a->kv_heads,
                                (uint64_t)(a->n_pages > 0 ? a->n_pages : 1)};
      const uint64_t str[3] = {(uint64_t)st * 2, (uint64_t)sh * 2, (uint64_t)(i ? a->v_stride_page : a->k_stride_page) * 2};
      const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
      rc = encode_tmap(tm, dt, 4, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    } else {
      const uint64_t dims[3] = {(uint64_t)D, (uint64_t)(a->tokens_k > 0 ? a->tokens_k : 1), (uint64_t)a->kv_heads};
      const uint64_t str[2] = {(uint64_t)st * 2, (uint64_t)sh * 2};
      const uint32_t box[3] = {64, 128, 1};
      rc = encode_tmap(tm, dt, 3, base, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (rc != TB200_OK) return rc;
  }
  p.o = a->o;
  p.lse = a->lse;
  p.status = status_ptr();
  if (!p.status) return TB200_ERR_CUDA;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  VarTile* pieces = reinterpret_cast<VarTile*>(ws + 32);
  VarSplit* splits = reinterpret_cast<VarSplit*>(ws + plan.off_splits);
  p.count = reinterpret_cast<VarCounters*>(ws);
  p.pieces = pieces;
  p.splits = splits;
  p.part_ml = reinterpret_cast<float2*>(ws + plan.off_ml);
  p.part_o = reinterpret_cast<float*>(ws + plan.off_o);
  p.page_table = a->page_table;
  p.table_stride = a->table_stride;
  p.o_stride_tok = a->o_stride_tok;
  p.o_stride_head = a->o_stride_head;
  p.heads = (int)a->heads;
  p.packs = plan.packs;
  p.gp = plan.gp;
  p.packs_per_kv = plan.packs / (int)a->kv_heads;
  p.page_size = a->page_size;
  p.box_rows = box_rows;
  p.n_pages = (int)a->n_pages;
  p.max_pages = (int)a->max_pages;
  p.no_page = p.n_pages > 0 ? p.n_pages : 1;
  p.causal = a->causal ? 1 : 0;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;

  ScheduleParams s;
  memset(&s, 0, sizeof(s));
  s.cu_q = a->cu_seqlens_q;
  s.cu_k = a->cu_seqlens_k;
  s.seq_lens = a->seq_lens;
  s.pieces = pieces;
  s.splits = splits;
  s.count = p.count;
  s.batch = (int)a->batch;
  s.tokens_q = (int)a->tokens_q;
  s.tokens_k = (int)a->tokens_k;
  s.packs = plan.packs;
  s.ctas = plan.ctas;
  s.max_pieces = (int)plan.max_pieces;
  s.max_splits = plan.max_split;
  s.max_parts = plan.max_parts;
  s.tile_tokens = plan.tile_tokens;
  s.group_tokens = plan.group_tokens;
  s.causal = p.causal;
  s.two_groups = D == 256 ? 0 : 1;
  s.paged = paged ? 1 : 0;
  s.max_len = (int)(a->max_pages * a->page_size);
  if (launch_overlapped(attention_varlen_schedule_kernel, dim3(1), 1024, 0, stream, s) != cudaSuccess) return TB200_ERR_CUDA;
  auto launch = paged ? (D == 256   ? launch_varlen<256, 1, true>
                         : D == 128 ? launch_varlen<128, 2, true> : launch_varlen<64, 2, true>)
                      : (D == 256   ? launch_varlen<256, 1, false>
                         : D == 128 ? launch_varlen<128, 2, false> : launch_varlen<64, 2, false>);
  return launch(p, f16, plan.ctas, plan.max_split, stream);
}
