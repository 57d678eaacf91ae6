// paged_dec.cuh -- attention of few new rows over a paged cache (decode): bf16, head_dim 64 or 128, any
// page size; definitions and work distribution in paged.cuh.
//
// Bound: HBM (each cached key and value is used by the group's rows only, g FLOP per byte).  A 128-row
// tcgen05 tile would be a few rows full and its chain of S, softmax and PV is longer.  Here a CTA's
// eight warps take the 16- or 32-key steps of its run in turn, rows as one 16-row
// m16n8k16 tile each, and every warp copies its next steps to shared memory ahead (cp.async,
// kDecStages deep, 192 KB per SM), across item boundaries too.  At an item's end the warps' rows
// meet in shared memory, row r merged by warp r % 8 while the others go on; of a split item the warp
// that writes a row's last piece joins the row's pieces, in their order.
// Measured, 32/8 heads of 128: 64 sequences of 500-8192 keys 130 us, 729 MB, 5.6 TB/s (SMs with equal work end
// between 94 and 127 us: their shares of the bandwidth differ); 4 of 65537-131071 keys with 64/8 heads 243 us,
// 6.5 TB/s; one of 2048 keys 10.5 us, all of it latency: launches, finding the run, page lookups, first keys, join.
// Probabilities are rounded to bf16 because the second product's operands are (the values, as cached): at most
// 2^-9 of each weight, their sum kept unrounded in fp32.  Against 64 bits an output is off by 2.3e-3 of its
// norm, where fp32 probabilities would give 1.7e-3, the output's own rounding.
#pragma once

#include "paged.cuh"

namespace beacon {

constexpr int kDecStages = 3, kDecWarps = 8, kDecRows = 16, kDecKt = 128;
// An item's start and end against 128 keys (90 sequences of 100-1000 tokens: cost 0 59 us, 1 47 us, 2 42 us).
constexpr int kDecItemCost = 2;
template <int D>
struct PagedDecCfg {
  static constexpr int KS = D == 64 ? 32 : 16;     // keys per step: 8 KB of keys and values
  static constexpr uint32_t ROW = D * 2;           // bytes of a key
  static constexpr uint32_t TILE = KS * ROW;       // a step's keys (or values)
  static constexpr uint32_t RING = kDecWarps * kDecStages * 2 * TILE;
  static constexpr int LDO = D + 8;                // merge rows, padded against bank conflicts
  static constexpr size_t SMEM_BYTES = (size_t)RING + kDecWarps * 8 * LDO * sizeof(float) + kDecWarps * 8 * sizeof(float2);
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8]: thread holds rows lane/4 (c0, c1) and lane/4 + 8 (c2, c3), columns
// 2 (lane % 4) and the next.
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
  v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return max_nan(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

template <int D>
__global__ void __launch_bounds__(256, 1) k_paged_attn_dec(const __nv_bfloat16* __restrict__ q,
                                                           const __nv_bfloat16* __restrict__ kc,
                                                           const __nv_bfloat16* __restrict__ vc, const PagedParams p) {
  using Cfg = PagedDecCfg<D>;
  constexpr int KS = Cfg::KS, NT = KS / 8, NH = KS / 16;
  constexpr int CH = D / 8;           // 16-byte chunks of a key
  constexpr int RPL = 32 / CH;        // keys that a warp copies per instruction
  constexpr int CPL = D / 32;         // columns per lane of a merged row
  extern __shared__ __align__(128) uint8_t dec_smem[];
  __shared__ uint64_t merge_full, merge_free;  // the merge buffer written, and read, by all eight warps
  __shared__ int abort_word;
  const int lane = (int)lane_id(), warp = (int)warp_id();
  const uint32_t ring = smem_u32(dec_smem) + warp * kDecStages * 2 * Cfg::TILE;
  float* mo = reinterpret_cast<float*>(dec_smem + Cfg::RING);                      // [8 warps][8 rows][LDO]
  float2* mml = reinterpret_cast<float2*>(mo + kDecWarps * 8 * Cfg::LDO);         // [8 warps][8 rows]
  const float scale_log2 = p.scale * 1.4426950408889634f;
  volatile int* abort_flag = &abort_word;
  if (threadIdx.x == 0) {
    mbar_init(&merge_full, kDecWarps);
    mbar_init(&merge_free, kDecWarps);
    abort_word = 0;
    fence_mbarrier_init();
  }
  __syncthreads();
  pdl_wait();

  // fragment addresses within a tile: chunk c of key r lies at chunk c ^ (r & 7) of its row
  const int kr = (lane & 7) + ((lane >> 4) << 3), kcb = (lane >> 3) & 1;  // K: keys x head dims
  const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vcb = lane >> 4;  // V, transposed on load
  const int cr = lane / CH, cc = lane % CH;                               // copies: key cr + RPL i, chunk cc

  PagedWalk<kDecKt> walk;  // every warp holds the same
  walk.start(p, (int)blockIdx.x, (int)gridDim.x);
  auto steps_of = [](const PagedItem& x) {  // steps of a piece, at least one
    const int key0 = x.a * kDecKt;
    return (min(x.b * kDecKt, max(x.kv, key0 + 1)) - key0 + KS - 1) / KS;
  };

  // The copies run ahead of the arithmetic on a walk of their own: the warp's next step is step fs of
  // piece fx, `off` the cache offset of its key (lane % KS), -1 for none.
  PagedWalk<kDecKt> fwalk = walk;
  PagedItem fx;
  int fs = 0, fn = 0;
  bool fon = true;
  long long off = -1;
  auto seek = [&]() {
#pragma unroll 1
    while (fon && fs >= fn) {
      fon = fwalk.next(p, fx);
      if (fon) {
        fs = warp;
        fn = steps_of(fx);
      }
    }
    const int key = fx.a * kDecKt + fs * KS + (lane & (KS - 1));
    off = fon && key < fx.kv ? paged_key(p.pg, fx.seq, fx.kvh, key) : -1;
  };
  int fstage = 0;
  auto fetch = [&]() {
    if (fon) {
      const uint32_t kt = ring + fstage * 2 * Cfg::TILE;
#pragma unroll
      for (int i = 0; i < KS / RPL; ++i) {
        const int r = cr + RPL * i;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t dst = kt + r * Cfg::ROW + ((cc ^ (r & 7)) << 4);
        const long long e = (o < 0 ? 0 : o) + cc * 8;
        cp_async16_or_zero(dst, kc + e, o >= 0);
        cp_async16_or_zero(dst + Cfg::TILE, vc + e, o >= 0);
      }
      fs += kDecWarps;
      seek();
    }
    cp_async_commit();
    fstage = fstage + 1 == kDecStages ? 0 : fstage + 1;
  };
  // query rows of this thread: lane / 4 and lane / 4 + 8 of the item
  uint32_t qf[D / 16][4];
  int lim[2];
  auto load_q = [&](const PagedItem& x) {
    const int rows = min(p.rpi, x.q_len * p.g - x.row0);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = lane / 4 + 8 * hf, fr = x.row0 + r;
      const bool have = r < rows;
      lim[hf] = have ? min(paged_limit(p, x, fr), x.kv) : 0;
      const __nv_bfloat16* qr = q + (long long)(x.q0 + (have ? fr / p.g : 0)) * p.q_stride +
                                ((long long)x.kvh * p.g + (have ? fr % p.g : 0)) * D + 2 * (lane & 3);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][hf] = have ? __ldg(reinterpret_cast<const uint32_t*>(qr + 16 * kk)) : 0u;
        qf[kk][2 + hf] = have ? __ldg(reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8)) : 0u;
      }
    }
  };
  // Writes row r of an item (whole) from its sum l relative to the maximum m (log2 units), CPL columns per lane.
  auto store_row = [&](const PagedItem& x, int r, float m, float l, const float (&o)[CPL]) {
    const int fr = x.row0 + r;
    const long long at = (long long)(x.q0 + fr / p.g) * p.Hq + (long long)x.kvh * p.g + fr % p.g;
    const bool sees = paged_limit(p, x, fr) > 0;
    const float inv = paged_inv(m, l);
    uint32_t w[CPL / 2];
#pragma unroll
    for (int e = 0; e < CPL; e += 2) w[e / 2] = !sees ? 0u : pack_bf16x2(o[e] * inv, o[e + 1] * inv);
    uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<__nv_bfloat16*>(p.out) + at * D + CPL * lane);
    if constexpr (CPL == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    else dst[0] = w[0];
    if (lane == 0 && p.lse != nullptr) p.lse[at] = paged_lse(m, __log2f(l));
  };

  PagedItem x;
  int stage = 0;
  uint32_t merges = 0;
  bool primed = false;
#pragma unroll 1
  while (walk.next(p, x)) {
    load_q(x);  // used after the first keys have come
    if (!primed) {
      primed = true;
      seek();
#pragma unroll 1
      for (int s = 0; s < kDecStages - 1; ++s) fetch();
    }
    float o[D / 8][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const int steps = steps_of(x);
    for (int s = warp; s < steps; s += kDecWarps) {
      __syncwarp();  // every lane has read the stage that the next copy overwrites
      fetch();
      cp_async_wait<kDecStages - 1>();
      __syncwarp();
      const uint32_t kt = ring + stage * 2 * Cfg::TILE, vt = kt + Cfg::TILE;
      stage = stage + 1 == kDecStages ? 0 : stage + 1;
      float sc[NT][4] = {};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          uint32_t b[4];
          ldsm_x4(b, kt + (kr + 16 * h) * Cfg::ROW + (((2 * kk + kcb) ^ (kr & 7)) << 4));
          mma_bf16(sc[2 * h], qf[kk], b[0], b[1]);
          mma_bf16(sc[2 * h + 1], qf[kk], b[2], b[3]);
        }
      const int k0 = x.a * kDecKt + s * KS + 2 * (lane & 3);
      uint32_t pf[NH][4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float v[2 * NT];
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 2 * NT; ++e) {
          v[e] = k0 + 8 * (e >> 1) + (e & 1) < lim[hf] ? sc[e >> 1][2 * hf + (e & 1)] * scale_log2 : -INFINITY;
          mx = max_nan(mx, v[e]);
        }
        mx = quad_max(mx);
        const float m_new = max_nan(m[hf], mx);
        // as long as the maximum grows by less than 2^8 the old one serves: O, l and P share it (a NaN is taken on)
        const bool need = !(m_new <= m[hf] + 8.0f);
        if (__any_sync(0xffffffffu, need)) {
          const float alpha = need ? ex2_approx(m[hf] - m_new) : 1.0f;
          if (need) m[hf] = m_new;
          l[hf] *= alpha;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * hf] *= alpha;
            o[n][2 * hf + 1] *= alpha;
          }
        }
        const float base = m[hf] == -INFINITY ? 0.0f : m[hf];
#pragma unroll
        for (int e = 0; e < 2 * NT; ++e) {
          v[e] = ex2_approx(v[e] - base);
          l[hf] += v[e];
        }
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          pf[h][hf] = pack_bf16x2(v[4 * h], v[4 * h + 1]);
          pf[h][2 + hf] = pack_bf16x2(v[4 * h + 2], v[4 * h + 3]);
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];
          ldsm_x4_t(b, vt + (vr + 16 * h) * Cfg::ROW + (((2 * n + vcb) ^ (vr & 7)) << 4));
          mma_bf16(o[2 * n], pf[h], b[0], b[1]);
          mma_bf16(o[2 * n + 1], pf[h], b[2], b[3]);
        }
    }
    const int rows = min(p.rpi, x.q_len * p.g - x.row0);
    const bool whole = x.a == 0 && x.b == x.n;
    const long long slot = paged_slot(x);
    const PagedPieces pc = paged_pieces(x);
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {  // rows r0 .. r0 + 7; the upper eight move down for their turn
      if (r0 == 8) {
        m[0] = m[1];
        l[0] = l[1];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] = o[n][2];
          o[n][1] = o[n][3];
        }
      }
      const float ls = quad_sum(l[0]);
      // every warp of the CTA arrives on both barriers for every merge, so these waits end
      mbar_wait(&merge_free, (merges & 1u) ^ 1u, abort_flag, kSitePagedMerge);
      float* mr = mo + (warp * 8 + lane / 4) * Cfg::LDO + 2 * (lane & 3);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(mr + 8 * n) = make_float2(o[n][0], o[n][1]);
      if ((lane & 3) == 0) mml[warp * 8 + lane / 4] = make_float2(m[0], ls);
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge_full);
      const int r = r0 + warp;
      float mx = -INFINITY, lt = 0.0f, ot[CPL] = {};
      if (r < rows) {  // row r: the warps' partial rows in warp order
        mbar_wait(&merge_full, merges & 1u, abort_flag, kSitePagedMerge);
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) mx = max_nan(mx, mml[w * 8 + warp].x);
        const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
          const float2 ml = mml[w * 8 + warp];
          const float wgt = ex2_approx(ml.x - base);
          lt = fmaf(ml.y, wgt, lt);
          const float* src = mo + (w * 8 + warp) * Cfg::LDO + CPL * lane;
          float sv[CPL];
          if constexpr (CPL == 4) *reinterpret_cast<float4*>(sv) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(sv) = *reinterpret_cast<const float2*>(src);
#pragma unroll
          for (int e = 0; e < CPL; ++e) ot[e] = fmaf(sv[e], wgt, ot[e]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&merge_free);
      ++merges;
      if (r >= rows) continue;
      if (whole) {
        store_row(x, r, mx, lt, ot);
        continue;
      }
      float* po = p.part_o + (slot * p.rpi + r) * D + CPL * lane;  // row-major slots: a warp holds one row
#pragma unroll
      for (int e = 0; e < CPL; ++e) po[e] = ot[e];
      if (lane == 0) p.part_ml[slot * p.rpi + r] = make_float2(mx, lt);
      if (!paged_last_piece(p, pc, r)) continue;
      // lane i weighs piece i (of 32 at a time); the pieces' rows then load side by side
      mx = -INFINITY;
      for (int i = lane; i < pc.n; i += 32) mx = max_nan(mx, __ldcg(&p.part_ml[pc.slot(i) * p.rpi + r]).x);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float base = mx == -INFINITY ? 0.0f : mx;
      lt = 0.0f;
#pragma unroll
      for (int e = 0; e < CPL; ++e) ot[e] = 0.0f;
#pragma unroll 1
      for (int i0 = 0; i0 < pc.n; i0 += 32) {
        const float2 ml = i0 + lane < pc.n ? __ldcg(&p.part_ml[pc.slot(i0 + lane) * p.rpi + r])
                                           : make_float2(-INFINITY, 0.0f);
        const float wl = ex2_approx(ml.x - base);
        lt += warp_sum(wl * ml.y);
        const int n = min(32, pc.n - i0);
#pragma unroll 1
        for (int i1 = 0; i1 < n; i1 += 8) {
          float v[8][CPL];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float* src = p.part_o + (pc.slot(i0 + min(i1 + i, n - 1)) * p.rpi + r) * D + CPL * lane;
            if constexpr (CPL == 4) *reinterpret_cast<float4*>(v[i]) = __ldcg(reinterpret_cast<const float4*>(src));
            else *reinterpret_cast<float2*>(v[i]) = __ldcg(reinterpret_cast<const float2*>(src));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float wgt = __shfl_sync(0xffffffffu, wl, min(i1 + i, 31));
            if (i1 + i < n) {
#pragma unroll
              for (int e = 0; e < CPL; ++e) ot[e] = fmaf(v[i][e], wgt, ot[e]);
            }
          }
        }
      }
      store_row(x, r, mx, lt, ot);
    }
  }
  cp_async_wait<0>();
}

}  // namespace beacon
