// paged_tc.cuh -- attention of new tokens over a paged cache on tcgen05 tensor cores (bf16, head_dim
// 64 or 128, pages of a multiple of 8 tokens; definitions and work distribution in paged.cuh).
//
// One CTA per SM walks its run of key tiles.  An item is a pair of 128-row query tiles (A, B) of one
// (sequence, KV head); a tile's rows are tpt = floor(128 / g) tokens x g heads of the group, fetched by
// one 4-D TMA box per 64 columns, so a group's heads share every K/V tile.  A 128-key tile is fetched
// page by page: lane i of the producer warp looks up its page one tile ahead and issues the box of
// its gcd(page_size, 128) keys; boxes past the sequence's keys take an out-of-range page and fill with
// zeros.  The slots between the last key and the end of its box may hold anything: the masked S
// columns are replaced, and the MMA warp overwrites those V rows with zeros before the tile's PV.
//
//   warp 0      producer (whole warp): the run's items (published in a ring), Q tiles, K ring
//   warp 2      producer of the V ring.  One producer of both let K(j+2) wait for the V stage that PV(j-1)
//               frees, so that a tile's S came late: 64 sequences of 500-8192 keys, 8 new tokens each,
//               32/8 heads of 128: 247 us with one, 153 us with two (144 now).
//   warp 1      TMEM allocator, MMA issuer:  S_A S_B | O_A += P_A V, S_A', O_B += P_B V, S_B' | ...
//   warps 4-7   softmax of tile A, warps 8-11 of tile B: one row per thread, fp32 statistics, P (bf16)
//               back into the S region of TMEM, O rescaled there when the maximum grows by over 2^8.
//               A pair's last key tile may be past tile A's last key: A then ends earlier.
//
// An item whose rows fit tile A is `dual`: B takes the same query tile over every other key tile, so
// that one tile's softmax still runs beside the other's products (a lone tile's chain of S, softmax
// and PV measured 2.2 us per 128 keys); at its end each of the two takes half of the columns.  The rows
// of an item in two pieces are joined by the warp that finishes the second one; k_paged_join joins
// those of items in more (one warp that reads 16 pieces took 45 us, the whole device a few).
//
// Bound: the softmax warps beside the tensor core.  2048 new tokens after 30720, 64/8 heads of 128: 1.73 ms =
// 1.23 PFLOP/s on a GPU that comes from idle, 2.0 ms in a loop under the power cap; tensor pipe active 68% of
// the cycles.  A 256-row step of 128 keys takes ~3.0k cycles, of them
// ~1.75k in softmax and ~1.2k waiting for the S that was issued behind the other tile's PV.  Short items pay
// ~7.5k cycles for their start and end (rows stored from registers, first softmax of both tiles at once):
// 16 sequences of 1-512 new tokens after 100-7500, 32/8 heads, 103-106 us from idle and 118 in a loop of calls,
// against 45 us of FLOPs.  Tiles, starts and ends, splits, the join and the launch at these costs make 80 to 85
// of them; where the rest goes has not been measured.  An item's end is fetched anew each time:
// unrolled by chunk it was slower (106 us against 103).
//
// P is rounded to bf16 because the operands of its product are of one type, the cached values': at most 2^-9
// of each weight; the row's sum l keeps the unrounded ones.
//
// TMEM: S_A [0,128), S_B [128,256), O_A [256,256+D), O_B [256+D,256+2D).
#pragma once

#include "attention.cuh"
#include "paged.cuh"

namespace beacon {

template <int D>
struct PagedTcCfg {
  static constexpr uint32_t Q_BYTES = 128 * D * 2;
  static constexpr uint32_t KV_BYTES = 128 * D * 2;
  static constexpr int STAGES = D == 64 ? 4 : 2;  // K and V tiles in flight: 64 KB each
  static constexpr size_t SMEM_BYTES = 1024 + 2 * (size_t)Q_BYTES + 2 * STAGES * (size_t)KV_BYTES + 1024 + 256 * sizeof(float2);
  static constexpr int THREADS = 384;
};

struct PagedTcParams {
  PagedParams p;
  float scale_log2;
  int tpt;        // tokens per query tile
  int box;        // keys per TMA box
};

enum : unsigned int {
  kSitePtcItem = 0x621,
  kSitePtcQ = 0x622,
  kSitePtcKv = 0x623,
  kSitePtcS = 0x624,
  kSitePtcP = 0x625,
  kSitePtcO = 0x626,
  kSitePtcClean = 0x627,
  kSitePtcDrain = 0x628,
  kSitePtcDual = 0x629,
};

constexpr int kPtcItems = 4;  // items published ahead
// Time of a key tile, of one of a dual item, and of an item's start and end (clock counts of every CTA of a
// launch over 16 sequences of 1-512 new tokens, heads of 128, fitted: 3390, 2330 and 7550 cycles).  Heads of 64
// take the same weights, which were not fitted there: the same sequences 95 us against a floor of 22.
constexpr int kPtcTile = 3, kPtcDualTile = 2, kPtcItemCost = 7;
struct PtcItem {
  int valid;
  int seq, kvh, tok0;  // sequence; KV head; first token row of the item in q
  int ntok;            // tokens from tok0 to the sequence's end
  int lim0;            // keys that token tok0 sees (tok0 + i: lim0 + i), or kv when not causal
  int kv;
  int a, b;            // key tiles [a, b)
  int end[2];          // the last key tile + 1 of tiles A, B within [a, b); <= a: none
  int dual;            // tiles A and B share the query tile and take key tiles a, a+2, .. and a+1, a+3, ..
  int slot;            // workspace slot of a partial piece, -1: the whole item
  PagedPieces pieces;  // the item's pieces
};
// Key tiles of an item's tile t in [a, b): first, step and count.
__device__ __forceinline__ int ptc_count(const PtcItem& x, int t) {
  return x.dual ? (x.b - x.a + 1 - t) / 2 : max(0, x.end[t] - x.a);
}

// 2^a for a pair of arguments on the FMA pipe: a = n + f, f in [-0.5, 0.5], a quartic in f fitted to 2^f by
// Lawson's iteration on the relative error (2.7e-6 in fp32), n added to the exponent.  The quartic, not
// the cubic of the training forward, because lse is returned to 1e-5.  Arguments below -126, -inf
// included, give less than 2^-125 instead of 0: masked keys add at most that to a row's sums.  NaN and
// +inf are lost here; the row's maximum keeps them (paged_inv).
__device__ __forceinline__ void exp2_poly4(float& r0, float& r1, float a0, float a1) {
  constexpr float kMagic = 12582912.0f;  // 1.5 x 2^23: adding it rounds to an integer
  a0 = fmaxf(a0, -126.0f);
  a1 = fmaxf(a1, -126.0f);
  float t0, t1, n0, n1, f0, f1, p0, p1;
  add2(t0, t1, a0, a1, kMagic, kMagic);
  add2(n0, n1, t0, t1, -kMagic, -kMagic);
  fma2(f0, f1, n0, n1, -1.0f, -1.0f, a0, a1);
  fma2(p0, p1, 9.5701022e-3f, 9.5701022e-3f, f0, f1, 5.5917859e-2f, 5.5917859e-2f);
  fma2(p0, p1, p0, p1, f0, f1, 2.4024744e-1f, 2.4024744e-1f);
  fma2(p0, p1, p0, p1, f0, f1, 6.9312179e-1f, 6.9312179e-1f);
  fma2(p0, p1, p0, p1, f0, f1, 9.9999928e-1f, 9.9999928e-1f);
  r0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  r1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}

// P = 2^(x scale - m) of one 128-key row into the 64 TMEM columns at `taddr` (bf16 pairs); returns the
// row's sum (fp32, before rounding).  Each 64-key half is handed to the MMA warp once stored.
__device__ __forceinline__ float ptc_softmax(const float* x, float scale_log2, float neg_m, uint32_t taddr,
                                             uint64_t* p_half) {
  float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t pk[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      float a0, a1, p0, p1;
      fma2(a0, a1, x[64 * c + 2 * e], x[64 * c + 2 * e + 1], scale_log2, scale_log2, neg_m, neg_m);
      if ((kPolyPairs >> (e & 7)) & 1u) {
        exp2_poly4(p0, p1, a0, a1);
      } else {
        p0 = ex2_approx(a0);
        p1 = ex2_approx(a1);
      }
      const int q = 2 * (e & 1);
      add2(ls[q], ls[q + 1], ls[q], ls[q + 1], p0, p1);
      pk[e] = pack_bf16x2(p0, p1);
    }
    tmem_st32(taddr + 32 * c, pk);
    tmem_wait_st();
    tc_fence_before();
    __syncwarp();
    if (lane_id() == 0) mbar_arrive(&p_half[c]);
  }
  return (ls[0] + ls[1]) + (ls[2] + ls[3]);
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Page of the box of keys that starts at `key`, or num_pages (outside the map: reads as zeros) when the
// sequence has no such key or the table names no page of the cache.
__device__ __forceinline__ int ptc_page(const PagedSeqs& g, int seq, int key, int kv) {
  if (key >= kv) return g.num_pages;
  const int page = __ldg(g.page_table + (long long)seq * g.table_stride + key / g.page_size);
  if (page >= 0 && page < g.num_pages) return page;
  record_fault(kFaultIndex, kSitePagedPage);
  return g.num_pages;
}

template <int D>
__global__ void __launch_bounds__(384, 1)
    k_paged_attn_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const PagedTcParams tp) {
  using Cfg = PagedTcCfg<D>;
  constexpr int ST = Cfg::STAGES;
  constexpr uint32_t LOG = ST == 2 ? 1 : 2;
  const PagedParams& p = tp.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * Cfg::Q_BYTES;
  uint8_t* sV = sK + ST * Cfg::KV_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * Cfg::KV_BYTES);
  uint64_t* k_full = bars;
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* q_full = v_empty + ST;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;   // [2] per tile
  uint64_t* p_full = s_full + 2;    // [2][2] per tile and 64-key half
  uint64_t* o_full = p_full + 4;    // [2]
  uint64_t* clean = o_full + 2;     // the MMA warp's lanes have zeroed a V tile's tail
  uint64_t* drain = clean + 1;
  uint64_t* dual_full = drain + 1;               // [4] per 32 rows of a dual item: A's and B's sums are final
  uint64_t* dual_free = dual_full + 4;           // [4] both have read the other's
  uint64_t* item_full = dual_free + 4;           // [kPtcItems]
  uint64_t* item_empty = item_full + kPtcItems;  // [kPtcItems] read by the MMA warp, the V producer and 8 softmax warps
  PtcItem* items = reinterpret_cast<PtcItem*>(item_empty + kPtcItems);
  float2* dual_ml = reinterpret_cast<float2*>(items + kPtcItems);  // [2][128] a dual item's (m, l)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dual_ml + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(clean, 32);
    mbar_init(drain, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&dual_full[i], 2);
      mbar_init(&dual_free[i], 2);
    }
    for (int i = 0; i < kPtcItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 10);
    }
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();  // everything above runs while the kernel before this one ends

  auto read_item = [&](int ci, PtcItem& x) -> bool {
    const int s = ci % kPtcItems;
    if (!mbar_wait(&item_full[s], (uint32_t)(ci / kPtcItems) & 1u, abort_flag, kSitePtcItem)) return false;
    x = items[s];
    return x.valid != 0;
  };

  // 128 x 72 + 256 x 216 = 384 x 168, the allocation the CTA is launched with
  if (warp < 4) {
    warpgroup_reg_dealloc<72>();
    if (warp == 0) {
      // -------------------------------------------------------------- producer
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        pdl_launch_dependents();
        p.heads[blockIdx.x] = PagedHead{};
      }
      PagedWalk<128, kPtcTile, kPtcDualTile> walk;
      walk.start(p, (int)blockIdx.x, (int)gridDim.x);
      const int nbox = 128 / tp.box;
      const uint32_t q_tile_bytes = (uint32_t)(tp.tpt * p.g) * 128u * (D / 64);
      uint32_t tk = 0, kissued = 0, kpar = 0, qissued = 0, qpar = 0;
      bool ok = true;
      for (int ci = 0; ok; ++ci) {
        PagedItem w{};
        const bool more = walk.next(p, w);
        PtcItem x{};
        x.valid = more ? 1 : 0;
        if (more) {
          const int t0 = w.row0 / p.g;
          x.seq = w.seq;
          x.kvh = w.kvh;
          x.tok0 = w.q0 + t0;
          x.ntok = w.q_len - t0;
          x.lim0 = p.causal ? w.kv - w.q_len + t0 + 1 : w.kv;
          x.kv = w.kv;
          x.slot = (w.a == 0 && w.b == w.n) ? -1 : paged_slot(w);
          x.a = w.a;
          x.b = w.b;
          x.pieces = paged_pieces(w);
          x.dual = x.ntok <= tp.tpt ? 1 : 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int last = min((t + 1) * tp.tpt, x.ntok) - 1;
            const int keys = p.causal ? max(0, x.lim0 + last) : x.kv;
            x.end[t] = t * tp.tpt < x.ntok ? min(x.b, max(1, (keys + 127) / 128)) : 0;
          }
        }
        const int is = ci % kPtcItems;
        ok = warp_wait(&item_empty[is], ((uint32_t)(ci / kPtcItems) & 1u) ^ 1u, abort_flag, kSitePtcItem);
        if (!ok) break;
        if (lane == 0) {
          items[is] = x;
          mbar_arrive(&item_full[is]);
          if (more && w.a == 0 && w.b < w.n && x.pieces.n > 2) p.heads[blockIdx.x] = paged_head(p, w);
        }
        if (!more) break;
        int page = (int)lane < nbox ? ptc_page(p.pg, w.seq, x.a * 128 + (int)lane * tp.box, w.kv) : 0;
        ok = warp_wait(q_empty, ((uint32_t)ci & 1u) ^ 1u, abort_flag, kSitePtcQ);
        if (!ok) break;
        if (lane == 0) {
          const int nt = x.end[1] > x.a ? 2 : 1, first = x.end[0] > x.a ? 0 : 1;
          mbar_arrive_expect_tx(q_full, (uint32_t)(nt - first) * q_tile_bytes);
          for (int t = first; t < nt; ++t)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(sQ + t * Cfg::Q_BYTES + c * 16384, &tmQ, q_full, c * 64, 0, x.tok0 + t * tp.tpt, x.kvh);
        }
        qissued = 1;
        qpar = (uint32_t)ci & 1u;
        for (int j = x.a; j < x.b; ++j, ++tk) {
          const uint32_t st = tk & (ST - 1), ph = (tk >> LOG) & 1u;
          const int key = j * 128 + (int)lane * tp.box, cur = page;
          if (j + 1 < x.b && (int)lane < nbox) page = ptc_page(p.pg, w.seq, key + 128, w.kv);
          const int row = key % p.pg.page_size;
          ok = warp_wait(&k_empty[st], ph ^ 1u, abort_flag, kSitePtcKv);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&k_full[st], Cfg::KV_BYTES);
          __syncwarp();
          if ((int)lane < nbox) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(sK + st * Cfg::KV_BYTES + c * 16384 + lane * tp.box * 128, &tmK, &k_full[st], c * 64, row,
                          x.kvh, cur);
          }
          kissued |= 1u << st;
          kpar = (kpar & ~(1u << st)) | (ph << st);
        }
      }
      if (!ok && lane == 0) {  // a wait gave up: the copies in flight land before the CTA may end
        volatile int no_abort = 0;
        if (qissued) mbar_wait(q_full, qpar, &no_abort, kSitePtcDrain);
        for (int s = 0; s < ST; ++s) {
          if (kissued & (1u << s)) mbar_wait(&k_full[s], (kpar >> s) & 1u, &no_abort, kSitePtcDrain);
        }
      }
    } else if (warp == 2) {
      // -------------------------------------------------------------- V producer
      const int nbox = 128 / tp.box;
      uint32_t tk = 0, vissued = 0, vpar = 0;
      bool ok = true;
      PtcItem x;
      for (int ci = 0; ok; ++ci) {
        const bool got = read_item(ci, x);
        if (!__all_sync(0xffffffffu, got)) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[ci % kPtcItems]);
        int page = (int)lane < nbox ? ptc_page(p.pg, x.seq, x.a * 128 + (int)lane * tp.box, x.kv) : 0;
        for (int j = x.a; j < x.b; ++j, ++tk) {
          const uint32_t st = tk & (ST - 1), ph = (tk >> LOG) & 1u;
          const int key = j * 128 + (int)lane * tp.box, cur = page;
          if (j + 1 < x.b && (int)lane < nbox) page = ptc_page(p.pg, x.seq, key + 128, x.kv);
          const int row = key % p.pg.page_size;
          ok = warp_wait(&v_empty[st], ph ^ 1u, abort_flag, kSitePtcKv);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&v_full[st], Cfg::KV_BYTES);
          __syncwarp();
          if ((int)lane < nbox) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(sV + st * Cfg::KV_BYTES + c * 16384 + lane * tp.box * 128, &tmV, &v_full[st], c * 64, row,
                          x.kvh, cur);
          }
          vissued |= 1u << st;
          vpar = (vpar & ~(1u << st)) | (ph << st);
        }
      }
      if (!ok && lane == 0) {
        volatile int no_abort = 0;
        for (int s = 0; s < ST; ++s)
          if (vissued & (1u << s)) mbar_wait(&v_full[s], (vpar >> s) & 1u, &no_abort, kSitePtcDrain);
      }
    } else if (warp == 1) {
      // -------------------------------------------------------------- MMA issuer
      const bool leader = elect_one();
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, false, false);
      constexpr uint32_t idesc_o = make_idesc_f16(128, D, false, true);
      const uint64_t q_desc = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = make_sdesc_sw128(smem_u32(sK), 16, 1024);
      const uint64_t v_desc = make_sdesc_sw128(smem_u32(sV), 128 * 128, 1024);
      auto issue_s = [&](int t, int qt, uint32_t k) {
        const uint64_t qd = sdesc_adv(q_desc, qt * Cfg::Q_BYTES), kd = sdesc_adv(k_desc, (k & (ST - 1)) * Cfg::KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * 16384 + (kk & 3) * 32;
          if (leader) umma_f16_ss(tmem + 128 * t, sdesc_adv(qd, off), sdesc_adv(kd, off), idesc_s, kk > 0 ? 1u : 0u);
        }
        if (leader) umma_commit(&s_full[t]);
      };
      uint32_t tk = 0, ns[2] = {0u, 0u}, nclean = 0;
      bool ok = true;
      PtcItem x;
      // per-lane waits inside an item, as in k_attn_fwd_tc: no warp collective until its end
      for (int ci = 0;; ++ci) {
        const bool got = ok && read_item(ci, x);
        if (!__all_sync(0xffffffffu, got)) break;
        const int n = x.b - x.a;
        const int tail = x.kv & 127;                                        // keys in the sequence's last tile
        const int dirty = tail % tp.box != 0 ? x.kv >> 7 : -1;              // the tile whose V rows need zeros
        const int dirty_end = tail + (tp.box - tail % tp.box);
        bool iok = lane_wait(q_full, (uint32_t)ci & 1u, abort_flag, kSitePtcQ) &&
                   lane_wait(&k_full[tk & (ST - 1)], (tk >> LOG) & 1u, abort_flag, kSitePtcKv);
        if (iok) {
          tc_fence_after();
          for (int t = 0; t < 2; ++t)
            if (x.dual ? t == 0 : x.end[t] > x.a) issue_s(t, t, tk);
          if (leader) umma_commit(&k_empty[tk & (ST - 1)]);
          if (n == 1 && leader) umma_commit(q_empty);
        }
        if (x.dual && n > 1 && iok) {
          iok = lane_wait(&k_full[(tk + 1u) & (ST - 1)], ((tk + 1u) >> LOG) & 1u, abort_flag, kSitePtcKv);
          if (iok) {
            tc_fence_after();
            issue_s(1, 0, tk + 1u);
            if (leader) umma_commit(&k_empty[(tk + 1u) & (ST - 1)]);
            if (n == 2 && leader) umma_commit(q_empty);
          }
        }
        for (int i = 0; i < n && iok; ++i) {
          const int j = x.a + i;
          const uint32_t tv = tk + (uint32_t)i, tn = tv + 1u;
          bool k_next = false;
          if (!lane_wait(&v_full[tv & (ST - 1)], (tv >> LOG) & 1u, abort_flag, kSitePtcKv)) { iok = false; break; }
          if (j == dirty) {
            uint8_t* vt = sV + (tv & (ST - 1)) * Cfg::KV_BYTES;
            const int chunks = (dirty_end - tail) * 8;
            for (int e = (int)lane; e < chunks * (D / 64); e += 32) {
              const int c = e / chunks, o = e - c * chunks;
              *reinterpret_cast<uint4*>(vt + c * 16384 + tail * 128 + o * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            mbar_arrive(clean);
            if (!lane_wait(clean, nclean & 1u, abort_flag, kSitePtcClean)) { iok = false; break; }
            ++nclean;
          }
          const uint64_t vd = sdesc_adv(v_desc, (tv & (ST - 1)) * Cfg::KV_BYTES);
          for (int t = 0; t < 2 && iok; ++t) {
            if (x.dual ? t != (i & 1) : j >= x.end[t]) continue;
            const uint32_t it = (uint32_t)(x.dual ? i >> 1 : i);  // the tile's how manieth key tile
            for (int hf = 0; hf < 2 && iok; ++hf) {
              if (!lane_wait(&p_full[2 * t + hf], (ns[t] + it) & 1u, abort_flag, kSitePtcP)) {
                iok = false;
                break;
              }
              tc_fence_after();
#pragma unroll
              for (int k4 = 0; k4 < 4; ++k4) {
                const int kk = 4 * hf + k4;
                if (leader)
                  umma_f16_ts(tmem + 256 + t * D, tmem + 128 * t + kk * 8, sdesc_adv(vd, kk * 2048), idesc_o,
                              (it > 0 || kk > 0) ? 1u : 0u);
              }
            }
            if (!iok) break;
            if (x.dual) {
              if (i + 2 >= n && leader) umma_commit(&o_full[t]);
              if (i + 2 < n) {
                const uint32_t t2 = tv + 2u;
                if (!lane_wait(&k_full[t2 & (ST - 1)], (t2 >> LOG) & 1u, abort_flag, kSitePtcKv)) { iok = false; break; }
                tc_fence_after();
                issue_s(t, 0, t2);
                if (leader) umma_commit(&k_empty[t2 & (ST - 1)]);
                if (i + 3 == n && leader) umma_commit(q_empty);
              }
              continue;
            }
            if (j == x.end[t] - 1 && leader) umma_commit(&o_full[t]);
            if (j + 1 < x.end[t]) {
              if (!k_next) {
                if (!lane_wait(&k_full[tn & (ST - 1)], (tn >> LOG) & 1u, abort_flag, kSitePtcKv)) { iok = false; break; }
                tc_fence_after();
                k_next = true;
              }
              issue_s(t, t, tn);
            }
          }
          if (!iok) break;
          if (leader) umma_commit(&v_empty[tv & (ST - 1)]);
          if (k_next && leader) umma_commit(&k_empty[tn & (ST - 1)]);
          if (!x.dual && i + 2 == n && leader) umma_commit(q_empty);
        }
        ok = iok;
        tk += (uint32_t)n;
        for (int t = 0; t < 2; ++t) ns[t] += (uint32_t)ptc_count(x, t);
        __syncwarp();
        if (ok && leader) mbar_arrive(&item_empty[ci % kPtcItems]);
      }
      if (leader) umma_commit(drain);
      volatile int no_abort = 0;
      warp_wait(drain, 0, &no_abort, kSitePtcDrain);
    }
  } else {
    warpgroup_reg_alloc<216>();
    // ---------------------------------------------------------------- softmax
    const int t = warp < 8 ? 0 : 1;
    const int r = (int)((warp & 3u) * 32 + lane);
    const uint32_t lane_base = ((warp & 3u) * 32u) << 16;
    const uint32_t s_col = 128 * t, o_col = 256 + t * D;
    const int rt = r / p.g;  // token of the tile
    const bool in_tile = rt < tp.tpt;
    const int head = r - rt * p.g;
    uint32_t ns = 0, no = 0, duals = 0;
    bool ok = true;
    for (int ci = 0; ok; ++ci) {
      PtcItem x;
      const bool more = __all_sync(0xffffffffu, read_item(ci, x));
      if (lane == 0) mbar_arrive(&item_empty[ci % kPtcItems]);
      if (!more) break;
      const int count = ptc_count(x, t), tok = (x.dual ? 0 : t * tp.tpt) + rt;
      const bool row_ok = in_tile && tok < x.ntok;
      // rows that are stored nowhere count as seeing every key, so that they do not force the masked path
      const int lim = !row_ok ? INT32_MAX : p.causal ? max(0, x.lim0 + tok) : x.kv;
      float m_used = -INFINITY, l = 0.0f;
      for (int i = 0; i < count; ++i) {
        const int j = x.dual ? x.a + t + 2 * i : x.a + i;
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], (ns + (uint32_t)i) & 1u, abort_flag, kSitePtcS))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int limit = lim - j * 128;
        if (!__all_sync(0xffffffffu, limit >= 128)) {
          // keys past the row's limit become -inf in TMEM, so that one softmax serves every tile: a second
          // one for masked tiles cost ~6k cycles of instruction fetch at its first use in a launch
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t u[32];
            tmem_ld32(tmem + lane_base + s_col + c, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] = c + e < limit ? u[e] : 0xff800000u;
            tmem_st32(tmem + lane_base + s_col + c, u);
          }
          tmem_wait_st();
        }
        uint32_t xu[128];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          tmem_ld32(tmem + lane_base + s_col + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&xu[32 * c]));
        tmem_wait_ld();
        float* xs = reinterpret_cast<float*>(xu);
        float m8[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) m8[u] = max_nan(xs[u], xs[8 + u]);
#pragma unroll
        for (int c = 16; c < 128; c += 16)
#pragma unroll
          for (int u = 0; u < 8; ++u) m8[u] = max3_nan(m8[u], xs[c + u], xs[c + 8 + u]);
        const float mx =
            max3_nan(max3_nan(m8[0], m8[1], m8[2]), max3_nan(m8[3], m8[4], m8[5]), max_nan(m8[6], m8[7])) *
            tp.scale_log2;
        const float m_new = max_nan(m_used, mx);
        if (i == 0) {
          m_used = m_new;
        } else {
          // a row without a key so far has O = 0 and m = -inf: 2^(-inf) = 0 rescales it; a NaN is taken on
          const bool need = !(m_new <= m_used + 8.0f);
          if (__any_sync(0xffffffffu, need)) {
            const float alpha = need ? ex2_approx(m_used - m_new) : 1.0f;
            if (need) {
              l *= alpha;
              m_used = m_new;
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t u[32];
              tmem_ld32(tmem + lane_base + o_col + c * 32, u);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * alpha);
              tmem_st32(tmem + lane_base + o_col + c * 32, u);
            }
          }
        }
        const float neg_m = m_used == -INFINITY ? 0.0f : -m_used;
        l += ptc_softmax(xs, tp.scale_log2, neg_m, tmem + lane_base + s_col, &p_full[2 * t]);
      }
      if (!ok) break;
      ns += (uint32_t)count;
      if (count > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&o_full[t], no & 1u, abort_flag, kSitePtcO))) {
          ok = false;
          break;
        }
        ++no;
        tc_fence_after();
      }
      // 32 columns of the row into a workspace slot
      auto store_part = [&](float4* dst, const uint32_t (&u)[32]) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dst[(long long)e * p.rpi] = make_float4(__uint_as_float(u[4 * e]), __uint_as_float(u[4 * e + 1]),
                                                  __uint_as_float(u[4 * e + 2]), __uint_as_float(u[4 * e + 3]));
      };
      // Dual: a row's two threads (same lanes of TMEM) hold sums over alternate key tiles.  Their statistics
      // cross through shared memory; then each finishes half of the row's columns.
      const uint32_t qd = warp & 3u;
      float w_a = 1.0f, w_b = 0.0f;
      int c0 = 0, c1 = D / 32;
      if (x.dual) {
        dual_ml[t * 128 + r] = make_float2(m_used, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dual_full[qd]);
        ok = warp_wait(&dual_full[qd], duals & 1u, abort_flag, kSitePtcDual);
        if (!ok) break;
        tc_fence_after();
        const float2 ml = dual_ml[(1 - t) * 128 + r];
        const float mx = max_nan(m_used, ml.x);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float w_own = ex2_approx(m_used - base), w_other = ex2_approx(ml.x - base);
        w_a = t == 0 ? w_own : w_other;
        w_b = t == 0 ? w_other : w_own;
        l = t == 0 ? fmaf(l, w_a, ml.y * w_b) : fmaf(ml.y, w_a, l * w_b);  // the same sum on both sides
        m_used = mx;
        c0 = t * (D / 64);
        c1 = c0 + D / 64;
      }
      const bool has = x.dual || count > 0;  // the tile saw keys of this piece
      // columns [32 c, 32 c + 32) of the row's O, relative to m_used (whole warp)
      auto load_o = [&](int c, uint32_t (&u)[32]) {
        if (!x.dual) {
          tmem_ld32(tmem + lane_base + o_col + c * 32, u);
          tmem_wait_ld();
          return;
        }
        tmem_ld32(tmem + lane_base + 256 + c * 32, u);
        if (x.b - x.a > 1) {
          uint32_t ub[32];
          tmem_ld32(tmem + lane_base + 256 + D + c * 32, ub);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            u[e] = __float_as_uint(fmaf(__uint_as_float(u[e]), w_a, __uint_as_float(ub[e]) * w_b));
        } else {
          tmem_wait_ld();  // A alone has had a key tile
        }
      };
      const long long at = (long long)(x.tok0 + tok) * p.Hq + (long long)x.kvh * p.g + head;
      __nv_bfloat16* orow = reinterpret_cast<__nv_bfloat16*>(p.out) + at * D;
      const bool out32 = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
      const bool none = lim <= 0;  // the row sees no key
      // stores 32 finished columns of the row, u inv
      auto store_o = [&](int c, const uint32_t (&u)[32], float inv) {
#pragma unroll
        for (int e = 0; e < 32; e += 16) {
          uint32_t wv[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            wv[i] = none ? 0u
                         : pack_bf16x2(__uint_as_float(u[e + 2 * i]) * inv, __uint_as_float(u[e + 2 * i + 1]) * inv);
          if (out32) {
            stg256(orow + c * 32 + e, wv[0], wv[1], wv[2], wv[3], wv[4], wv[5], wv[6], wv[7]);
          } else {
            *reinterpret_cast<uint4*>(orow + c * 32 + e) = make_uint4(wv[0], wv[1], wv[2], wv[3]);
            *reinterpret_cast<uint4*>(orow + c * 32 + e + 8) = make_uint4(wv[4], wv[5], wv[6], wv[7]);
          }
        }
      };
      const bool any_row = __any_sync(0xffffffffu, row_ok);
      const bool lse_row = p.lse != nullptr && !(x.dual && t == 1);
      if (x.slot < 0) {
        if (!has) continue;  // a tile B without rows
        const float inv = paged_inv(m_used, l);
#pragma unroll 1
        for (int c = c0; c < c1 && any_row; ++c) {
          uint32_t u[32];
          load_o(c, u);
          if (row_ok) store_o(c, u, inv);
        }
        if (row_ok && lse_row) p.lse[at] = paged_lse(m_used, __log2f(l));
      } else if (any_row) {
        const int row = (x.dual ? 0 : t * tp.tpt * p.g) + r;  // row of the item
        // statistics of the row; B keeps its own copy of a dual item's, in rows that the item does not have
        const int ml_row = row + (x.dual ? t * tp.tpt * p.g : 0);
        const long long own = (long long)x.slot * p.rpi + ml_row;
        // mostly the other piece, the first of its run, was written long ago
        bool last = x.pieces.n == 2 && paged_others_done(p, x.pieces, (int)warp - 4);
        if (!last) {
          if (has) {
#pragma unroll 1
            for (int c = c0; c < c1; ++c) {
              uint32_t u[32];
              load_o(c, u);
              if (row_ok) store_part(paged_part(p, x.slot, 8 * c, row), u);
            }
          }
          // without a key tile here: m = -inf, and its O, not written, is not read
          if (row_ok) p.part_ml[own] = make_float2(m_used, l);
          last = x.pieces.n == 2 && paged_last_piece(p, x.pieces, (int)warp - 4);
        }
        if (last) {
          const int mine = x.a > 0 ? 1 : 0;  // this piece is the item's first or second
          const long long that = x.pieces.slot(1 - mine);
          const float2 ml = row_ok ? __ldcg(&p.part_ml[that * p.rpi + ml_row]) : make_float2(-INFINITY, 0.0f);
          const float mx = max_nan(m_used, ml.x);
          const bool read = row_ok && ml.x != -INFINITY;
          const float base = mx == -INFINITY ? 0.0f : mx;
          const float w_mine = ex2_approx(m_used - base), w_that = ex2_approx(ml.x - base);
          const float lt = mine ? fmaf(l, w_mine, ml.y * w_that) : fmaf(ml.y, w_that, l * w_mine);
          const float inv = paged_inv(mx, lt);
          const float4* src = paged_part(p, that, 8 * c0, row);
          float4 v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = read ? __ldcg(src + (long long)e * p.rpi) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
          for (int c = c0; c < c1; ++c) {
            uint32_t u[32];
            if (has) {
              load_o(c, u);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) u[e] = 0u;
            }
            const float* f = reinterpret_cast<const float*>(v);
#pragma unroll
            for (int e = 0; e < 32; ++e) {  // first piece, then second: the same sum whichever joins
              const float a = __uint_as_float(u[e]);
              u[e] = __float_as_uint(mine ? fmaf(a, w_mine, f[e] * w_that) : fmaf(f[e], w_that, a * w_mine));
            }
            if (c + 1 < c1) {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                v[e] = read ? __ldcg(src + (long long)(8 * (c + 1 - c0) + e) * p.rpi) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (row_ok) store_o(c, u, inv);
          }
          if (row_ok && lse_row) p.lse[at] = paged_lse(mx, __log2f(lt));
        }
        __syncwarp();
      }
      tc_fence_before();
      if (x.dual) {  // the other tile's thread has read this one's O and statistics
        __syncwarp();
        if (lane == 0) mbar_arrive(&dual_free[qd]);
        ok = warp_wait(&dual_free[qd], duals & 1u, abort_flag, kSitePtcDual);
        if (!ok) break;
        ++duals;
        tc_fence_after();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace beacon
