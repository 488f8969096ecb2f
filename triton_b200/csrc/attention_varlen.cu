// Flash-attention forward over packed sequences of different lengths, with grouped heads; keys and values packed too, or
// in the pages of a cache. O = softmax(Q K^T * sm_scale [+ causal mask]) V per sequence, base-2 log-sum-exp per row.
//
// The pipeline is that of attention.cu (warp 0 TMA loads, warp 1 issues every tcgen05.mma, two softmax warpgroups of 128
// query rows that alternate on the tensor pipe; S and P in tensor memory, O rescaled only when the running maximum grew
// by more than 2^8). What differs:
//   rows      A group's 128 rows are 128 / gp consecutive tokens x gp query heads of one kv head (gp = the largest power
//             of two in heads / kv_heads): one box of a 4-D tensor map (column, head of the pack, token, pack). A tile so
//             covers fewer tokens, which wastes less on short sequences and on the causal diagonal, and K / V are read
//             once per pack instead of once per head.
//   schedule  attention_varlen_schedule_kernel turns the sequence offsets into a list of tiles, the longest KV walks
//             first; the lengths never pass through the host. CTAs take tiles from the list in rounds of alternating
//             direction (the first round dealt from the long end, the second back, ...), which evens out their sums.
//   tails     The last KV block of a sequence runs into the next sequence's rows (or into whatever a page holds). Scores
//             there are replaced by -inf, so K's content is irrelevant; V's is not (0 * NaN), so warps 2 and 3 overwrite
//             those rows of the V tile with zeros in shared memory before the P V product may read it.
//   half      A tile whose tokens fit the first group (short sequences, ends) leaves the second group out.
//   pages     A KV block is 128 / r boxes of r = gcd(page size, 128) rows; the lanes of the load warp look up and issue one
//             page each. A page outside the pool is loaded from behind its end, which reads as zeros.
#include <string.h>

#include "attention_common.cuh"
#include "common.cuh"
#include "host_common.h"

namespace tb200 {

static constexpr int VAR_THREADS = 384;
static constexpr int VAR_BN = 128;      // kv rows per block
static constexpr int VAR_MAX_STAGES = 4;
static constexpr float VAR_RESCALE_THRESHOLD = 8.0f;

// One tile of the schedule (32 bytes): n_tok tokens from packed row tok0 on; diag = the last key position that token 0
// of the tile sees under a causal mask; n0 / n1 = KV blocks of the first / second group (n1 = 0: no tokens in it).
struct VarTile {
  int tok0, n_tok, kv_len, kv_first, diag, n0, n1, pad;
};
static_assert(sizeof(VarTile) == 32, "two 16-byte loads");

struct VarlenParams {
  CUtensorMap tmq;       // (D, gp, tokens, packs), box (64, gp, 128 / gp, 1), 128-byte swizzle
  CUtensorMap tmk, tmv;  // packed: (D, tokens, kv heads), box (64, 128, 1); pages: (D, page rows, kv heads, pages), box (64, r, 1, 1)
  void* o;
  float* lse;
  int* status;
  const VarTile* tiles;
  const int* n_tiles;
  const int32_t* page_table;
  long long table_stride, o_stride_tok, o_stride_head;
  int heads, packs, lgp, packs_per_kv;
  int page_size, box_rows, n_pages, max_pages;
  int no_page;  // first page coordinate behind the pool: reads as zeros
  int causal;
  float scale_log2;
};

struct ScheduleParams {
  const int32_t *cu_q, *cu_k, *seq_lens;
  VarTile* tiles;
  int* n_tiles;
  int batch, tokens_q, tokens_k, cap, tile_tokens, group_tokens, causal, two_groups, paged;
  int max_len;  // pages: what the page table can hold
};

struct SeqExtent {
  int q0, q_len, k_len, k_first;
};
__device__ __forceinline__ SeqExtent seq_extent(const ScheduleParams& p, int b) {
  SeqExtent s;
  s.q0 = max(p.cu_q[b], 0);
  s.q_len = max(min(p.cu_q[b + 1], p.tokens_q) - s.q0, 0);
  if (p.paged) {
    s.k_len = min(max(p.seq_lens[b], 0), p.max_len);
    s.k_first = b;
  } else {
    s.k_first = min(max(p.cu_k[b], 0), p.tokens_k);
    s.k_len = max(min(p.cu_k[b + 1], p.tokens_k) - s.k_first, 0);
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
  t.pad = 0;
  return t;
}

// One block. A counting sort of all tiles by their KV blocks, most first; one warp per sequence at a time. The order
// inside a bucket is left to the atomics: it decides which CTA runs a tile, not what the tile computes.
static constexpr int SCHED_BUCKETS = 1024;
__global__ void __launch_bounds__(1024) attention_varlen_schedule_kernel(const ScheduleParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  __shared__ int count[SCHED_BUCKETS];
  __shared__ int warp_sum[32];
  __shared__ int most;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  count[threadIdx.x] = 0;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  int mine = 0;
  for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
    const SeqExtent s = seq_extent(p, b);
    if (s.q_len > 0) mine = max(mine, s.k_len);
  }
  atomicMax(&most, mine);
  __syncthreads();
  const int top = 2 * ((most + VAR_BN - 1) / VAR_BN) + 2;
  int shift = 0;
  while ((top >> shift) >= SCHED_BUCKETS) ++shift;
  auto each_tile = [&](auto&& f) {
    for (int b = warp; b < p.batch; b += 32) {
      const SeqExtent s = seq_extent(p, b);
      const int n = (s.q_len + p.tile_tokens - 1) / p.tile_tokens;
      for (int i = lane; i < n; i += 32) {
        const VarTile t = make_tile(p, s, i);
        f(t, SCHED_BUCKETS - 1 - min((t.n0 + t.n1) >> shift, SCHED_BUCKETS - 1));
      }
    }
  };
  each_tile([&](const VarTile&, int bucket) { atomicAdd(&count[bucket], 1); });
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
  if (threadIdx.x == 0) *p.n_tiles = min(warp_sum[31], p.cap);
  __syncthreads();
  each_tile([&](const VarTile& t, int bucket) {
    const int at = atomicAdd(&count[bucket], 1);
    if (at < p.cap) {
      reinterpret_cast<int4*>(p.tiles + at)[0] = make_int4(t.tok0, t.n_tok, t.kv_len, t.kv_first);
      reinterpret_cast<int4*>(p.tiles + at)[1] = make_int4(t.diag, t.n0, t.n1, 0);
    }
  });
}

// G = query groups per CTA: 2, or 1 for head dim 256 (tiles of 64 KB, an accumulator of 256 columns).
template <int D, int G>
struct VarSmem {
  static constexpr int TILE_BYTES = 128 * D * 2;
  static constexpr int KV_STAGES = G == 2 ? VAR_MAX_STAGES : 2;
  static constexpr int Q_OFFSET = 0;
  static constexpr int KV_OFFSET = G * TILE_BYTES;
  static constexpr int BAR_OFFSET = KV_OFFSET + KV_STAGES * TILE_BYTES;
  static constexpr int NUM_BARS = 4 + 2 * VAR_MAX_STAGES + 16;
  static constexpr int TOTAL = BAR_OFFSET + NUM_BARS * 8 + 16 + 1024;
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* tmap, uint64_t* bar, int c0, int c1, int c2,
                                            int c3, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
      "l"(policy)
      : "memory");
}

// Rounds of alternating direction through the list (see the head of the file).
__device__ __forceinline__ int var_unit(int round) {
  const int at = (round & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x;
  return round * (int)gridDim.x + at;
}
__device__ __forceinline__ VarTile var_tile(const VarlenParams& p, int unit) {
  const int4* src = reinterpret_cast<const int4*>(p.tiles + unit / p.packs);
  const int4 a = src[0], b = src[1];
  return VarTile{a.x, a.y, a.z, a.w, b.x, b.y, b.z, 0};
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
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFFSET);
  uint64_t* q_full = bars;                       // [2]
  uint64_t* q_empty = bars + 2;                  // [2]
  uint64_t* kv_full = bars + 4;                  // [KV]
  uint64_t* kv_empty = kv_full + VAR_MAX_STAGES; // [KV]
  uint64_t* s_full = kv_empty + VAR_MAX_STAGES;  // [2] MMA -> softmax: S_g ready
  uint64_t* p_full = s_full + 2;                 // [2][4] softmax -> MMA: 32-column chunk c of P_g written (128 arrivals)
  uint64_t* pv_done = p_full + 8;                // [2] MMA -> softmax: last PV_g of the tile complete
  uint64_t* o_free = pv_done + 2;                // [2] softmax -> MMA: O_g read out (128 arrivals)
  uint64_t* v_dirty = o_free + 2;                // MMA -> warps 2, 3: the V tile ahead holds rows behind the sequence's end
  uint64_t* v_clean = v_dirty + 1;               // warps 2, 3 -> MMA: those rows are zero
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_clean + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tmq);
    tma_prefetch_desc(&p.tmk);
    tma_prefetch_desc(&p.tmv);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      for (int c = 0; c < 4; ++c) mbar_init(&p_full[i * 4 + c], 128);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_free[i], 128);
    }
    for (int i = 0; i < VAR_MAX_STAGES; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(v_dirty, 1);
    mbar_init(v_clean, 2);
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
  const int units = *p.n_tiles * p.packs;
  const uint32_t smem_a = smem_u32(smem);
  const int group_tokens = 128 >> p.lgp;

  if (warp == 0) {
    // ------------------------------------------------------------------ loader (whole warp; lane 0 waits and counts)
    reg_dealloc<104>();
    const uint64_t pol_q = policy_evict_first();
    const uint64_t pol_kv = policy_evict_last();
    const int n_boxes = PAGED ? VAR_BN / p.box_rows : 1;
    uint32_t pos = 0, tc0 = 0, tc1 = 0;
    bool ok = true;
    auto load_q = [&](int g, const VarTile& t, int pack) {
      if (lane == 0) {
        mbar_expect_tx(&q_full[g], L::TILE_BYTES);
#pragma unroll
        for (int b = 0; b < DBOX; ++b)
          tma_load_4d(smem + L::Q_OFFSET + g * L::TILE_BYTES + b * BOX_BYTES, &p.tmq, &q_full[g], b * 64, 0,
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
        go = mbar_wait(&kv_empty[stage], ((pos / KV_STAGES) & 1) ^ 1, status, WAIT_SMEM_EMPTY);
        if (go) mbar_expect_tx(&kv_full[stage], L::TILE_BYTES);
      }
      go = __shfl_sync(0xffffffffu, (int)go, 0) != 0;
      if (!go) return false;
      uint8_t* dst = smem + L::KV_OFFSET + stage * L::TILE_BYTES;
      if (PAGED) {
        if (lane < n_boxes) {
          const int in_page = (j * VAR_BN + lane * p.box_rows) % p.page_size;
#pragma unroll
          for (int b = 0; b < DBOX; ++b)
            tma_load_4d(dst + b * BOX_BYTES + lane * p.box_rows * 128, tm, &kv_full[stage], b * 64, in_page, kvh, page,
                        pol_kv);
        }
      } else if (lane == 0) {
#pragma unroll
        for (int b = 0; b < DBOX; ++b)
          tma_load_3d(dst + b * BOX_BYTES, tm, &kv_full[stage], b * 64, t.kv_first + j * VAR_BN, kvh, pol_kv);
      }
      ++pos;
      return true;
    };
    auto wait_q = [&](int g, uint32_t count) -> bool {
      bool go = true;
      if (lane == 0) go = mbar_wait(&q_empty[g], (count & 1) ^ 1, status, WAIT_SMEM_EMPTY);
      return __shfl_sync(0xffffffffu, (int)go, 0) != 0;
    };
    for (int r = 0; ok; ++r) {
      const int unit = var_unit(r);
      if (r * (int)gridDim.x >= units) break;
      if (unit >= units) continue;
      const VarTile t = var_tile(p, unit);
      const int pack = unit % p.packs, kvh = pack / p.packs_per_kv;
      const int n = max(t.n0, t.n1);
      int page = page_of(t, 0);
      if (!wait_q(0, tc0++)) break;
      load_q(0, t, pack);
      if (!load_kv(&p.tmk, t, kvh, 0, page)) break;
      if (TWO && t.n1 > 0) {
        if (!wait_q(1, tc1++)) break;
        load_q(1, t, pack);
      }
      if (!load_kv(&p.tmv, t, kvh, 0, page)) break;
      for (int j = 1; j < n && ok; ++j) {
        page = page_of(t, j);
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
        umma_commit(&s_full[g]);
      };
      // PV_g in four slices of 32 keys, each as soon as the softmax has published that chunk of P_g
      auto issue_pv = [&](int g, uint32_t vstage, uint32_t accum, uint32_t iph, bool ready, bool last) -> bool {
        const uint64_t vd = vdesc0 + (uint64_t)((vstage * L::TILE_BYTES) >> 4);
        const uint32_t d_o = tmem_base + O_COL0 + g * D;
        const uint32_t a_p = tmem_base + g * S_COLS;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (!ready && !mbar_wait(&p_full[g * 4 + c], iph, status, WAIT_ATTN)) return false;
          tc_fence_after_sync();
          if (c < 3) ready = mbar_test(&p_full[g * 4 + c + 1], iph);  // probe ahead of this slice's MMAs
#pragma unroll
          for (int k = 2 * c; k < 2 * (c + 1); ++k)
            umma_f16_ts(d_o, a_p + k * 8, vd + (uint64_t)((k * 16 * 128) >> 4), idp, (k > 0) ? 1u : accum);
        }
        if (last) umma_commit(&pv_done[g]);
        return true;
      };
      auto advance = [&]() {
        if (++kvs == KV_STAGES) {
          kvs = 0;
          kvph ^= 1;
        }
      };

      for (int r = 0; ok; ++r) {
        const int unit = var_unit(r);
        if (r * (int)gridDim.x >= units) break;
        if (unit >= units) continue;
        const VarTile t = var_tile(p, unit);
        const int n0 = t.n0, n1 = TWO ? t.n1 : 0, n = max(n0, n1);
        const bool both = TWO && n1 > 0;
        const uint32_t tph0 = tc0++ & 1, tph1 = tc1 & 1;
        if (both) ++tc1;
        // prologue: S_g(0) = Q_g K(0)^T
        const uint32_t kcur = kvs, kcur_ph = kvph;
        advance();
        if (!mbar_wait(&q_full[0], tph0, status, WAIT_ATTN)) break;
        if (!mbar_wait(&kv_full[kcur], kcur_ph, status, WAIT_SMEM_FULL)) break;
        tc_fence_after_sync();
        issue_qk(0, kcur);
        if (both) {
          if (!mbar_wait(&q_full[1], tph1, status, WAIT_ATTN)) break;
          tc_fence_after_sync();
          issue_qk(1, kcur);
        }
        umma_commit(&kv_empty[kcur]);
        // A walk that ends behind the sequence's end: its last V tile is cleaned before use. The helpers are told once
        // the full phase before that tile's in its ring stage has been seen here, so their wait cannot mistake an
        // earlier phase for it, and not again before they have answered.
        const bool tail = n * VAR_BN > t.kv_len;
        if (tail && n == 1) mbar_arrive(v_dirty);
        // the second group's diagonal lies at most 128 keys behind the first one's: n0 is n1 or n1 - 1
        if (n0 == 1) umma_commit(&q_empty[0]);
        if (both && n1 == 1) umma_commit(&q_empty[1]);
        for (int j = 0; j < n; ++j) {
          const uint32_t iph0 = it0 & 1, iph1 = it1 & 1;
          const bool act0 = j < n0, more0 = j + 1 < n0, more = j + 1 < n;
          const uint32_t vcur = kvs, vcur_ph = kvph;
          advance();
          uint32_t knext = 0, knext_ph = 0;
          if (more) {
            knext = kvs;
            knext_ph = kvph;
            advance();
          }
          if (!mbar_wait(&kv_full[vcur], vcur_ph, status, WAIT_SMEM_FULL)) { ok = false; break; }
          if (tail && j == n - 2) mbar_arrive(v_dirty);
          if (tail && j == n - 1) {
            if (!mbar_wait(v_clean, clean++ & 1, status, WAIT_ATTN)) { ok = false; break; }
            tc_fence_after_sync();
          }
          const bool k_ready = more && mbar_test(&kv_full[knext], knext_ph);
          if (act0) {
            if (j == 0 && !mbar_wait(&o_free[0], tph0 ^ 1, status, WAIT_ATTN)) { ok = false; break; }
            if (!issue_pv(0, vcur, j > 0 ? 1u : 0u, iph0, mbar_test(&p_full[0], iph0), !more0)) { ok = false; break; }
            ++it0;
          }
          bool p1_ready = false;
          if (more) {
            if (!k_ready && !mbar_wait(&kv_full[knext], knext_ph, status, WAIT_SMEM_FULL)) { ok = false; break; }
            tc_fence_after_sync();
            if (both) p1_ready = mbar_test(&p_full[4], iph1);
            if (more0) {
              issue_qk(0, knext);
              if (j + 2 == n0) umma_commit(&q_empty[0]);
            }
          }
          if (both) {
            if (j == 0 && !mbar_wait(&o_free[1], tph1 ^ 1, status, WAIT_ATTN)) { ok = false; break; }
            if (!issue_pv(1, vcur, j > 0 ? 1u : 0u, iph1, p1_ready, !more)) { ok = false; break; }
            ++it1;
          }
          umma_commit(&kv_empty[vcur]);
          if (more) {
            if (both) issue_qk(1, knext);
            umma_commit(&kv_empty[knext]);
            if (both && j + 2 == n1) umma_commit(&q_empty[1]);
          }
        }
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ V rows behind the end of a sequence
    reg_dealloc<104>();
    uint32_t pos = 0, told = 0;
    for (int r = 0;; ++r) {
      const int unit = var_unit(r);
      if (r * (int)gridDim.x >= units) break;
      if (unit >= units) continue;
      const VarTile t = var_tile(p, unit);
      const int n = max(t.n0, t.n1);
      if (n * VAR_BN > t.kv_len) {  // only the last block of a walk can reach behind the end
        const uint32_t at = pos + 2 * (n - 1) + 1, stage = at % KV_STAGES;
        if (!mbar_wait(v_dirty, told++ & 1, status, WAIT_ATTN)) break;
        if (!mbar_wait(&kv_full[stage], (at / KV_STAGES) & 1, status, WAIT_SMEM_FULL)) break;
        const int first = max(t.kv_len - (n - 1) * VAR_BN, 0);  // row r of a box lies in its bytes [128 r, 128 r + 128)
        const int chunks = (VAR_BN - first) * 8;
        for (int i = (warp - 2) * 32 + lane; i < chunks * DBOX; i += 64) {
          const int box = i / chunks, c = i - box * chunks;
          *reinterpret_cast<uint4*>(smem + L::KV_OFFSET + stage * L::TILE_BYTES + box * BOX_BYTES + first * 128 + c * 16) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
      }
      pos += 2 * n;
    }
  } else {
    // ------------------------------------------------------------------ softmax / correction / epilogue
    reg_alloc<192>();
    const int g = (warp - 4) >> 2;
    const int q = warp & 3;
    const int row = q * 32 + lane;                       // row of the group
    const int tok_row = g * group_tokens + (row >> p.lgp);  // token of the tile
    const int head_row = row & ((1 << p.lgp) - 1);          // head of the pack
    const uint32_t lane_off = (uint32_t)(q * 32) << 16;
    const uint32_t t_s = tmem_base + lane_off + g * S_COLS;
    const uint32_t t_o = tmem_base + lane_off + O_COL0 + g * D;
    const float scale = p.scale_log2;
    uint32_t it = 0, tcount = 0;
    bool ok = true;
    for (int r = 0; ok && (TWO || g == 0); ++r) {
      const int unit = var_unit(r);
      if (r * (int)gridDim.x >= units) break;
      if (unit >= units) continue;
      const VarTile t = var_tile(p, unit);
      const int n = g == 0 ? t.n0 : t.n1;
      if (n == 0) continue;
      float m = -INFINITY, l = 0.f;
      const int last = p.causal ? min(t.kv_len - 1, t.diag + tok_row) : t.kv_len - 1;  // last visible key of this row
      const int safe = p.causal ? min(t.kv_len - 1, t.diag + g * group_tokens) : t.kv_len - 1;  // ... of the group's first row
      for (int j = 0; j < n; ++j, ++it) {
        if (!mbar_wait(&s_full[g], it & 1, status, WAIT_ATTN)) { ok = false; break; }
        tc_fence_after_sync();
        const int k0 = j * VAR_BN;
        uint32_t sv[128];
        tmem_ld_row32<0>(t_s, sv);
        tmem_ld_row32<32>(t_s + 32, sv);
        tmem_ld_row32<64>(t_s + 64, sv);
        tmem_ld_row32<96>(t_s + 96, sv);
        tmem_ld_wait();
        if (k0 + VAR_BN - 1 > safe) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (k0 + i > last) sv[i] = 0xff800000u;  // -inf: contributes exp2(-inf) = 0
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
            mbar_arrive(&p_full[g * 4 + (c >> 5) - 1]);
          }
          tmem_st_32x32b_x16(t_s + (c >> 1), pk);
        }
        float sum_lo, sum_hi;
        unpack2(sum2, sum_lo, sum_hi);
        l += sum_lo + sum_hi;
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&p_full[g * 4 + 3]);
      }
      if (!ok) break;
      if (!mbar_wait(&pv_done[g], tcount++ & 1, status, WAIT_ATTN)) break;
      tc_fence_after_sync();
      const float inv_l = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no visible key: zeros; NaN stays NaN
      const bool valid = tok_row < t.n_tok;
      const long long token = t.tok0 + tok_row;
      const int head = (unit % p.packs << p.lgp) + head_row;
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
            mbar_arrive(&o_free[g]);
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

template <int D, int G, bool PAGED>
static int launch_varlen(const VarlenParams& p, bool f16, int grid, cudaStream_t stream) {
  using L = VarSmem<D, G>;
  static_assert(L::TOTAL <= 232448, "shared memory budget");
  auto kfn = f16 ? attention_varlen_kernel<D, true, G, PAGED> : attention_varlen_kernel<D, false, G, PAGED>;
  if (cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL) != cudaSuccess)
    return TB200_ERR_CUDA;
  // starts while the schedule is being made: barriers and tensor memory are set up by the time it is there
  return cuda_err(launch_overlapped(kfn, dim3((unsigned)grid), VAR_THREADS, L::TOTAL, stream, p));
}

struct VarPlan {
  int lgp, tile_tokens, group_tokens;
  int64_t cap;
};
static VarPlan var_plan(const tb200_attention_varlen_args* a) {
  VarPlan v;
  const int64_t group = a->heads / a->kv_heads;
  v.lgp = 0;
  while (v.lgp < 7 && group % (2 << v.lgp) == 0) ++v.lgp;
  v.group_tokens = 128 >> v.lgp;
  v.tile_tokens = (a->head_dim == 256 ? 1 : 2) * v.group_tokens;
  v.cap = a->tokens_q / v.tile_tokens + a->batch;  // every sequence ends in at most one tile that is not full
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
  return 32 + (size_t)var_plan(a).cap * sizeof(VarTile);
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
  if (a->tokens_q > (1 << 30) || a->tokens_k > (1 << 30) || a->batch > (1 << 30) || a->heads > (1 << 16) ||
      a->n_pages > (1 << 30) || a->max_pages > (1 << 30) || a->max_pages * a->page_size > (1 << 30))
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
  const int packs = (int)(a->heads >> plan.lgp);
  if (plan.cap * packs > INT32_MAX / 2) return TB200_ERR_UNSUPPORTED;
  if (!a->workspace || a->workspace_bytes < tb200_attention_varlen_workspace_bytes(a) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 31))
    return TB200_ERR_BAD_ARG;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int sms = sm_count();
  if (sms <= 0) return TB200_ERR_CUDA;

  VarlenParams p;
  memset(&p, 0, sizeof(p));
  const int D = a->head_dim;
  const bool f16 = a->dtype == TB200_F16;
  const CUtensorMapDataType dt = f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  {
    const uint64_t gp = 1ull << plan.lgp;
    const uint64_t dims[4] = {(uint64_t)D, gp, (uint64_t)a->tokens_q, (uint64_t)packs};
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
  int* n_tiles = static_cast<int*>(a->workspace);
  VarTile* tiles = reinterpret_cast<VarTile*>(static_cast<uint8_t*>(a->workspace) + 32);
  p.tiles = tiles;
  p.n_tiles = n_tiles;
  p.page_table = a->page_table;
  p.table_stride = a->table_stride;
  p.o_stride_tok = a->o_stride_tok;
  p.o_stride_head = a->o_stride_head;
  p.heads = (int)a->heads;
  p.packs = packs;
  p.lgp = plan.lgp;
  p.packs_per_kv = packs / (int)a->kv_heads;
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
  s.tiles = tiles;
  s.n_tiles = n_tiles;
  s.batch = (int)a->batch;
  s.tokens_q = (int)a->tokens_q;
  s.tokens_k = (int)a->tokens_k;
  s.cap = (int)plan.cap;
  s.tile_tokens = plan.tile_tokens;
  s.group_tokens = plan.group_tokens;
  s.causal = p.causal;
  s.two_groups = D == 256 ? 0 : 1;
  s.paged = paged ? 1 : 0;
  s.max_len = (int)(a->max_pages * a->page_size);
  attention_varlen_schedule_kernel<<<1, 1024, 0, stream>>>(s);
  if (cudaGetLastError() != cudaSuccess) return TB200_ERR_CUDA;

  const int64_t most = plan.cap * packs;
  const int grid = most < sms ? (int)most : sms;
  if (paged)
    return D == 256 ? launch_varlen<256, 1, true>(p, f16, grid, stream)
           : D == 128 ? launch_varlen<128, 2, true>(p, f16, grid, stream) : launch_varlen<64, 2, true>(p, f16, grid, stream);
  return D == 256 ? launch_varlen<256, 1, false>(p, f16, grid, stream)
         : D == 128 ? launch_varlen<128, 2, false>(p, f16, grid, stream) : launch_varlen<64, 2, false>(p, f16, grid, stream);
}
