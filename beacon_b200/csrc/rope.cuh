// rope.cuh -- RMS norm of each query and key head and the position rotation in one pass,
// between the QKV projection (rows of (Hq + 2 Hkv) heads per token) and attention:
// head-major tensors for training, token-major queries and a paged key/value cache for
// serving, and the backward of the training form.
//
// One head x[D] of a token at position t, gain g[D] (optional), rot rotated dims (even):
//   r = sqrt(mean x^2 + eps), z = g x / r,
//   y_a = z_a c_i - z_b s_i, y_b = z_b c_i + z_a s_i, i < rot / 2,  y_d = z_d for d >= rot,
// with (a, b) = (i, i + rot/2), or (2i, 2i+1) interleaved, and (c_i, s_i) = the table's row t
// (rot/2 cosines, then rot/2 sines).  Without a gain z = x (rotation only).  Backward, dz the
// rotation of dy by the opposite angle:
//   dg += sum dz x / r,  e = g dz,  dx = e / r - x sum(e x) / (D r^3)   (dx = dz without a gain).
// Bound: HBM (each head is read once and written once; ~10 FLOP per element).
#pragma once

#include "elementwise.cuh"
#include "sm100.cuh"

namespace beacon {

// A batch of sequences whose keys and values live in pages: sequence s owns the new tokens
// [cu_q[s], cu_q[s+1]) of the token-major tensors and kv_lens[s] tokens of the cache, the
// new ones included and last; its j-th token sits in slot j % page_size of page
// page_table[s][j / page_size].
struct PagedSeqs {
  const int* cu_q;        // [seqs + 1]
  const int* kv_lens;     // [seqs]
  const int* page_table;  // [seqs, table_stride]
  long long table_stride;
  int seqs, max_pages, num_pages, page_size;
  long long page_stride, head_stride, token_stride;  // of both caches, in elements
};

struct RopeParams {
  int Hq, Hkv, D, rot, interleaved;
  float eps;
  long long tokens;
  int seq;                 // head-major forms: tokens per batch entry
  const float* table;      // [table_positions, rot]
  long long table_positions;
  const int* positions;    // [tokens] or null (token % seq, or the token's place in its sequence)
  long long ld;            // elements between token rows of qkv (and of dqkv: ld_out)
  long long ld_out;
  PagedSeqs pg;            // paged form
};

enum : unsigned int {
  kSiteRopePosition = 0x601,  // a position outside the table, or before the sequence's start
  kSiteRopePage = 0x602,      // a page index outside the cache, a token past the page table, or a cu_q that decreases
};

// Number of i in [1, n] with cu[i] <= t (the sequence that owns token t; n: none does).
// Whole warp, 32-way: two dependent loads up to 1024 sequences.
__device__ __forceinline__ int warp_owner(const int* __restrict__ cu, int n, int t) {
  const int lane = (int)lane_id();
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const bool on = (long long)lane * step < n;
    const int at = min((lane + 1) * step, n);
    const bool le = on && __ldg(cu + lo + at) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    const int active = __popc(__ballot_sync(0xffffffffu, on));
    const int skip = min(c * step, n);
    n = c < active ? min((c + 1) * step, n) - skip - 1 : 0;
    lo += skip;
  }
  return lo;
}

// Where a token goes: its rotation row, and the element offset of its slot for KV head 0.  32-bit
// divisions (a token count fits an int): the 64-bit ones were most of the kernels' instructions.
struct TokenPlace {
  bool on;         // the token belongs to a sequence (paged form)
  int pos;         // table row, -1: none (the head rows are written as zeros)
  int b, s;        // head-major form: batch entry and place in the sequence
  long long slot;  // paged form: cache offset of (page, head 0, token), -1: nowhere
};
// The sequence that the last token belonged to: a warp's tokens ascend, and in a prompt the next one is
// mostly of the same sequence, so that only its page is left to look up.
struct TokenSeq {
  int s = -1, first = 0, end = 0, kv = 0;
};
template <bool PAGED>
__device__ __forceinline__ TokenPlace token_place(const RopeParams& p, int t, TokenSeq& q) {
  TokenPlace w{true, 0, 0, 0, -1};
  if constexpr (PAGED) {
    const PagedSeqs& g = p.pg;
    if (q.s < 0 || t < q.first || t >= q.end) {
      q.s = warp_owner(g.cu_q, g.seqs, t);
      if (q.s < g.seqs) {
        q.first = __ldg(g.cu_q + q.s);
        q.end = __ldg(g.cu_q + q.s + 1);
        q.kv = max(0, __ldg(g.kv_lens + q.s));
      }
      if (q.s >= g.seqs || t < q.first || t >= q.end) {
        if (q.s < g.seqs && t >= q.end && lane_id() == 0) record_fault(kFaultIndex, kSiteRopePage);  // cu_q decreases
        q.s = -1;
        w.on = false;
        return w;
      }
    }
    const int s = q.s, at = q.kv - (q.end - t);
    w.pos = at;
    if (at >= 0) {
      const int pi = (int)((unsigned)at / (unsigned)g.page_size);
      int page = -1;
      if (pi < g.max_pages) page = __ldg(g.page_table + (long long)s * g.table_stride + pi);
      if (page >= 0 && page < g.num_pages)
        w.slot = (long long)page * g.page_stride + (long long)(at - pi * g.page_size) * g.token_stride;
      else if (lane_id() == 0)
        record_fault(kFaultIndex, kSiteRopePage);
    }
  } else {
    w.b = (int)((unsigned)t / (unsigned)p.seq);
    w.s = t - w.b * p.seq;
    w.pos = w.s;
  }
  if (p.positions != nullptr && w.pos >= 0) w.pos = __ldg(p.positions + t);
  if (w.pos < 0 || w.pos >= p.table_positions) {
    if (lane_id() == 0) record_fault(kFaultIndex, kSiteRopePosition);
    w.pos = -1;
  }
  return w;
}

// Destination of head h of kind 0 (query), 1 (key) or 2 (value) of token t; null: not written.
template <typename T, bool PAGED>
__device__ __forceinline__ T* head_out(const RopeParams& p, const TokenPlace& w, int t, int kind, int h, T* q, T* k,
                                       T* v) {
  T* base = kind == 0 ? q : kind == 1 ? k : v;
  if constexpr (PAGED) {
    if (kind == 0) return base + ((long long)t * p.Hq + h) * p.D;
    return w.slot < 0 ? nullptr : base + w.slot + (long long)h * p.pg.head_stride;
  } else {
    if (base == nullptr) return nullptr;
    return base + ((long long)(w.b * (kind == 0 ? p.Hq : p.Hkv) + h) * p.seq + w.s) * p.D;
  }
}

// Rotation partner of element d (d < rot) and the pair's index; first: d is the pair's first member.
__device__ __forceinline__ void rope_pair(int d, int rot, int interleaved, int& i, int& partner, bool& first) {
  const int half = rot >> 1;
  if (interleaved) {
    i = d >> 1;
    partner = d ^ 1;
    first = (d & 1) == 0;
  } else {
    first = d < half;
    i = first ? d : d - half;
    partner = first ? d + half : d - half;
  }
}

// Any head_dim up to kRopeMaxDim, any alignment: one warp per (token, head), element by element,
// the row read a second time from L1 for the rotation.
constexpr int kRopeMaxDim = 256;
template <typename T, bool PAGED>
__global__ void __launch_bounds__(256) k_qk_norm_rope_any(T* __restrict__ q, T* __restrict__ k, T* __restrict__ v,
                                                          const T* __restrict__ qkv, const T* __restrict__ q_gain,
                                                          const T* __restrict__ k_gain, const RopeParams p) {
  const int lane = (int)lane_id();
  const int heads = p.Hq + 2 * p.Hkv;
  const long long n = p.tokens * heads, warps = (long long)gridDim.x * (blockDim.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  for (long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; u < n; u += warps) {
    const long long t = u / heads;
    const int h = (int)(u - t * heads);
    TokenSeq seq;
    const TokenPlace w = token_place<PAGED>(p, (int)t, seq);
    if (!w.on) continue;
    const int kind = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2;
    T* o = head_out<T, PAGED>(p, w, (int)t, kind, kind == 0 ? h : kind == 1 ? h - p.Hq : h - p.Hq - p.Hkv, q, k, v);
    if (o == nullptr) continue;
    const T* x = qkv + t * p.ld + (long long)h * p.D;
    if (kind == 2) {
      for (int d = lane; d < p.D; d += 32) o[d] = x[d];
      continue;
    }
    const T* g = kind == 0 ? q_gain : k_gain;
    float inv = 1.0f;
    if (g != nullptr) {
      float ss = 0.0f;
      for (int d = lane; d < p.D; d += 32) ss = fmaf(ldf(x + d), ldf(x + d), ss);
      inv = 1.0f / sqrtf(warp_sum(ss) / (float)p.D + p.eps);
    }
    const float* tab = p.table + (long long)w.pos * p.rot;
    for (int d = lane; d < p.D; d += 32) {
      float y = w.pos < 0 ? 0.0f : ldf(x + d) * inv * (g != nullptr ? ldf(g + d) : 1.0f);
      if (w.pos >= 0 && d < p.rot) {
        int i, e;
        bool first;
        rope_pair(d, p.rot, p.interleaved, i, e, first);
        const float z = ldf(x + e) * inv * (g != nullptr ? ldf(g + e) : 1.0f);
        const float c = __ldg(tab + i), s = __ldg(tab + (p.rot >> 1) + i);
        y = first ? y * c - z * s : y * c + z * s;
      }
      stf(o + d, y);
    }
  }
}

// Backward, same mapping; part: [gridDim.x, 2, D] partial sums of dq_gain and dk_gain (fp32), each
// CTA's warps added in warp order, or null.
template <typename T>
__global__ void __launch_bounds__(256) k_qk_norm_rope_bwd_any(T* __restrict__ dqkv, float* __restrict__ part,
                                                              const T* __restrict__ dq, const T* __restrict__ dk,
                                                              const T* __restrict__ dv, const T* __restrict__ qkv,
                                                              const T* __restrict__ q_gain,
                                                              const T* __restrict__ k_gain, const RopeParams p) {
  __shared__ float red[8][kRopeMaxDim];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = (int)lane_id(), warp = (int)warp_id();
  const int heads = p.Hq + 2 * p.Hkv;
  const long long n = p.tokens * heads, warps = (long long)gridDim.x * (blockDim.x >> 5);
  float acc[2][kRopeMaxDim / 32] = {};
  for (long long u = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5; u < n; u += warps) {
    const long long t = u / heads;
    const int h = (int)(u - t * heads);
    TokenSeq seq;
    const TokenPlace w = token_place<false>(p, (int)t, seq);
    const int kind = h < p.Hq ? 0 : h < p.Hq + p.Hkv ? 1 : 2;
    const T* dy = head_out<const T, false>(p, w, (int)t, kind, kind == 0 ? h : kind == 1 ? h - p.Hq : h - p.Hq - p.Hkv, dq,
                                           dk, dv);
    if (dy == nullptr) continue;
    T* o = dqkv + t * p.ld_out + (long long)h * p.D;
    if (kind == 2) {
      for (int d = lane; d < p.D; d += 32) o[d] = dy[d];
      continue;
    }
    const T* x = qkv + t * p.ld + (long long)h * p.D;
    const T* g = kind == 0 ? q_gain : k_gain;
    const float* tab = p.table + (long long)w.pos * p.rot;
    float dz[kRopeMaxDim / 32], ss = 0.0f, ex = 0.0f;
#pragma unroll
    for (int j = 0; j < kRopeMaxDim / 32; ++j) {
      const int d = lane + 32 * j;
      dz[j] = 0.0f;
      if (d >= p.D || w.pos < 0) continue;
      dz[j] = ldf(dy + d);
      if (d < p.rot) {
        int i, e;
        bool first;
        rope_pair(d, p.rot, p.interleaved, i, e, first);
        const float c = __ldg(tab + i), s = __ldg(tab + (p.rot >> 1) + i);
        dz[j] = first ? dz[j] * c + ldf(dy + e) * s : dz[j] * c - ldf(dy + e) * s;
      }
      if (g != nullptr) {
        const float xv = ldf(x + d);
        ss = fmaf(xv, xv, ss);
        ex = fmaf(dz[j] * ldf(g + d), xv, ex);
      }
    }
    float inv = 1.0f, back = 0.0f;
    if (g != nullptr && w.pos >= 0) {
      ss = warp_sum(ss);
      ex = warp_sum(ex);
      inv = 1.0f / sqrtf(ss / (float)p.D + p.eps);
      back = ex * inv * inv / (float)p.D;
    }
#pragma unroll
    for (int j = 0; j < kRopeMaxDim / 32; ++j) {
      const int d = lane + 32 * j;
      if (d >= p.D) continue;
      if (g == nullptr) {
        stf(o + d, dz[j]);
      } else {
        const float xv = ldf(x + d);
        if (w.pos >= 0) {
          const float add = dz[j] * xv * inv;
          if (kind == 0) acc[0][j] += add;
          else acc[1][j] += add;
        }
        stf(o + d, w.pos < 0 ? 0.0f : inv * (dz[j] * ldf(g + d) - xv * back));
      }
    }
  }
  if (part == nullptr) return;
  for (int kind = 0; kind < 2; ++kind) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRopeMaxDim / 32; ++j) red[warp][lane + 32 * j] = kind == 0 ? acc[0][j] : acc[1][j];
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
      float s = 0.0f;
      for (int w = 0; w < 8; ++w) s += red[w][d];
      part[((long long)blockIdx.x * 2 + kind) * p.D + d] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// Vectorised forms: head_dim 64, 128 or 256, rot % 16 == 0, 16-byte aligned rows.
//
// A head takes D/16 lanes, each holding two 8-element chunks rot/2 apart, so that both members of a
// rotated pair sit in one lane (halves or interleaved) and the only exchange is the sum over the
// head's lanes; the lanes behind rot/16 hold the pass-through elements the same way.  A warp keeps
// one batch of U * 32/(D/16) heads of one kind (query, key or value) for every token it visits: its
// gains stay in registers and a token's cosines and sines are loaded once per batch.  Each lane
// copies its chunks of the next kRopeStages - 1 tokens to shared memory ahead (cp.async; only the
// lane itself reads them, so nothing synchronises): the bytes in flight do not cost registers.
// Two stages, two CTAs of eight warps per SM: a third CTA spilled, and equal runs of one kind of head per
// warp scattered the streams (forward 72 -> 86 us).
// Measured: forward, 8192 tokens of 32 + 32 + 32 heads of 128, bf16: 71.6 us, 403 MB, 5.6 TB/s; a copy with
// this access pattern alone 69 us.  Prompts of 10k tokens, 64 / 8 heads, into pages of 64: 81.5 us, 4.9 TB/s.
// What is left: issue slots (41-53% used) and 16 warps per SM to cover the rest with.
// ---------------------------------------------------------------------------
constexpr int kRopeStages = 2;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes, or zeros where `have` is false (nothing is read then).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A lane's staging area: N chunks of 8 elements per stage, its 16-byte pieces 512 bytes apart (a
// warp's pieces lie side by side, without bank conflicts).
template <typename T, int N>
struct RopeStage {
  static constexpr int PIECES = (int)sizeof(T) / 2;
  static constexpr uint32_t BYTES = N * PIECES * 512;  // per warp and stage
  uint32_t base;
  __device__ __forceinline__ RopeStage(void* smem, int warp)
      : base(smem_u32(smem) + warp * kRopeStages * BYTES + lane_id() * 16u) {}
  __device__ __forceinline__ void fetch(int stage, int chunk, const T* src) const {
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
      cp_async16(base + stage * BYTES + (chunk * PIECES + k) * 512, reinterpret_cast<const uint4*>(src) + k);
  }
  __device__ __forceinline__ void read(int stage, int chunk, Raw8<T>& r) const {
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.u[k].x), "=r"(r.u[k].y), "=r"(r.u[k].z), "=r"(r.u[k].w)
                   : "r"(base + stage * BYTES + (chunk * PIECES + k) * 512)
                   : "memory");
  }
  __device__ __forceinline__ void zero(int chunk, int n) const {
    for (int s = 0; s < kRopeStages; ++s)
      for (int k = 0; k < n * PIECES; ++k)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + s * BYTES + (chunk * PIECES + k) * 512),
                     "r"(0)
                     : "memory");
  }
};

struct RopeBatches {
  int nq, nk;  // batches of query heads, of key heads (value heads: as many as key heads)
  __host__ __device__ int total() const { return nq + 2 * nk; }
};

// Elements [e0, e0+8) and [e1, e1+8) of a head are lane l's; turns: they are rotated.
template <int D>
struct RopeLane {
  int sub, l, e0, e1;  // head of the warp's 32/(D/16), lane within it
  bool turns;
  __device__ __forceinline__ explicit RopeLane(int rot) {
    constexpr int LPH = D / 16;
    const int lane = (int)lane_id();
    l = lane % LPH;
    sub = lane / LPH;
    turns = l < rot / 16;
    e0 = turns ? 8 * l : rot + 8 * (l - rot / 16);
    e1 = e0 + (turns ? rot / 2 : (D - rot) / 2);
  }
  // Sum over the head's lanes.
  __device__ __forceinline__ float sum(float v) const {
#pragma unroll
    for (int o = D / 32; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  // Cosines and sines of the lane's eight pairs (1, 0 where nothing turns).  Halves: pair i joins
  // elements i of the two chunks; interleaved: pairs 0-3 lie in the first chunk, 4-7 in the second.
  __device__ __forceinline__ void turn(const RopeParams& p, int pos, float (&c)[8], float (&s)[8]) const {
    if (!turns || pos < 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = 1.0f;
        s[i] = 0.0f;
      }
      return;
    }
    const float* tab = p.table + (long long)pos * p.rot;
    const int i0 = p.interleaved ? e0 >> 1 : e0, i1 = p.interleaved ? e1 >> 1 : e0 + 4;
    const int half = p.rot >> 1;
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(tab + i0));
    const float4 c1 = __ldg(reinterpret_cast<const float4*>(tab + i1));
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(tab + half + i0));
    const float4 s1 = __ldg(reinterpret_cast<const float4*>(tab + half + i1));
    c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
    s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
  }
};

// Eight-element arithmetic in f32x2 instructions: issue slots, not bandwidth, are what these kernels run
// short of (scalar forms measured 2-5% slower).
__device__ __forceinline__ void mul8(float (&r)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    mul2(r[i], r[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
}
__device__ __forceinline__ void scale8(float (&r)[8], const float (&a)[8], float w) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    mul2(r[i], r[i + 1], a[i], a[i + 1], w, w);
}
__device__ __forceinline__ void fma8(float (&r)[8], const float (&a)[8], const float (&b)[8], const float (&c)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    fma2(r[i], r[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
}
__device__ __forceinline__ void fmaw8(float (&r)[8], const float (&a)[8], float w, const float (&c)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    fma2(r[i], r[i + 1], a[i], a[i + 1], w, w, c[i], c[i + 1]);
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8], const float (&c)[8],
                                      const float (&d)[8]) {
  float x0 = 0.0f, x1 = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    fma2(x0, x1, a[i], a[i + 1], b[i], b[i + 1], x0, x1);
    fma2(y0, y1, c[i], c[i + 1], d[i], d[i + 1], y0, y1);
  }
  return (x0 + x1) + (y0 + y1);
}

// A lane's part of a linear map of pairs: element i of the first chunk becomes pa[i] a[i] + qa[i] a'[i], a' its
// partner (the second chunk's element i, or its neighbour when interleaved); the second chunk likewise.
struct RopeMap {
  float pa[8], qa[8], pb[8], qb[8];
  // rotation by the angles (c, s) after scaling element-wise by (ga, gb)
  __device__ __forceinline__ void set(const float (&c)[8], const float (&s)[8], const float (&ga)[8],
                                      const float (&gb)[8], bool interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (interleaved) {
        const int j = i >> 1;
        pa[i] = ga[i] * c[j];
        qa[i] = (i & 1) ? ga[i ^ 1] * s[j] : -ga[i ^ 1] * s[j];
        pb[i] = gb[i] * c[4 + j];
        qb[i] = (i & 1) ? gb[i ^ 1] * s[4 + j] : -gb[i ^ 1] * s[4 + j];
      } else {
        pa[i] = ga[i] * c[i];
        qa[i] = -gb[i] * s[i];
        pb[i] = gb[i] * c[i];
        qb[i] = ga[i] * s[i];
      }
    }
  }
  __device__ __forceinline__ void apply(float (&a)[8], float (&b)[8], bool turns, bool interleaved) const {
    float u[8], w[8];
    mul8(u, a, pa);
    mul8(w, b, pb);
    if (turns) {
      if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u[i] = fmaf(a[i ^ 1], qa[i], u[i]);
          w[i] = fmaf(b[i ^ 1], qb[i], w[i]);
        }
      } else {
        fma8(u, b, qa, u);
        fma8(w, a, qb, w);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = u[i];
      b[i] = w[i];
    }
  }
};

// (a, b) = the lane's 16 elements turned back by the pairs' angles.
__device__ __forceinline__ void rope_back(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8],
                                          bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& x = i < 4 ? a[2 * i] : b[2 * i - 8];
      float& y = i < 4 ? a[2 * i + 1] : b[2 * i - 7];
      const float u = x * c[i] + y * s[i], w = y * c[i] - x * s[i];
      x = u;
      y = w;
    }
  } else {
    float u[8], w[8], t[8];
    mul8(u, b, s);
    mul8(w, a, s);
    mul8(t, b, c);
    fma8(a, a, c, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = t[i] - w[i];
  }
}

template <typename T>
__device__ __forceinline__ void straw(T* p, const Raw8<T>& r) {
#pragma unroll
  for (int k = 0; k < (int)(sizeof(T) / 2); ++k) reinterpret_cast<uint4*>(p)[k] = r.u[k];
}

// The warp's batch: kind 0 query, 1 key, 2 value heads; its lane's first head, the kind's count and
// its first head's column in a token row.
template <int D, int U>
struct RopeWork {
  int kind, h0, count, col, step, t0;
  bool on;
  __device__ __forceinline__ RopeWork(const RopeParams& p, const RopeBatches& nb, int sub) {
    const unsigned n = (unsigned)nb.total(), gw = blockIdx.x * (blockDim.x >> 5) + warp_id();
    const unsigned warps = gridDim.x * (blockDim.x >> 5);
    const int b = (int)(gw % n);
    step = (int)(warps / n);
    t0 = (int)(gw / n);
    on = gw < n * (unsigned)step;  // no work for warps beyond a whole number of rounds
    kind = b < nb.nq ? 0 : b < nb.nq + nb.nk ? 1 : 2;
    h0 = (kind == 0 ? b : kind == 1 ? b - nb.nq : b - nb.nq - nb.nk) * (U * 32 / (D / 16)) + sub;
    count = kind == 0 ? p.Hq : p.Hkv;
    col = kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.Hkv;
  }
};

// First element of head 0 of a kind for a token in the output of the forward (or the gradients that
// the backward reads), and the elements between heads; null: nothing is written.
template <typename T, int D, bool PAGED>
__device__ __forceinline__ T* rope_heads(const RopeParams& p, const TokenPlace& w, int t, int kind, int count, T* base,
                                         long long& stride) {
  if constexpr (PAGED) {
    stride = kind == 0 ? D : p.pg.head_stride;
    if (kind == 0) return base + (long long)t * p.Hq * D;
    return w.slot < 0 ? nullptr : base + w.slot;
  } else {
    stride = (long long)p.seq * D;
    return base == nullptr ? nullptr : base + ((long long)w.b * count * p.seq + w.s) * D;
  }
}

template <typename T, int D, int U, bool PAGED>
__global__ void __launch_bounds__(256, 2) k_qk_norm_rope_vec(T* __restrict__ q, T* __restrict__ k, T* __restrict__ v,
                                                             const T* __restrict__ qkv, const T* __restrict__ q_gain,
                                                             const T* __restrict__ k_gain, const RopeParams p,
                                                             const RopeBatches nb) {
  constexpr int HPW = 32 / (D / 16);
  extern __shared__ __align__(16) uint8_t rope_smem[];
  const RopeLane<D> ln(p.rot);
  const RopeWork<D, U> w(p, nb, ln.sub);
  pdl_launch_dependents();
  if (!w.on) return;
  pdl_wait();
  const RopeStage<T, 2 * U> st(rope_smem, (int)warp_id());
  const T* gain = w.kind == 0 ? q_gain : w.kind == 1 ? k_gain : nullptr;
  auto fetch = [&](long long t, int stage) {  // 64 bits: t runs past the last token
    if (t < p.tokens) {
      const T* row = qkv + t * p.ld + (long long)w.col * D;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = w.h0 + u * HPW;
        if (h >= w.count) continue;
        st.fetch(stage, 2 * u, row + (long long)h * D + ln.e0);
        st.fetch(stage, 2 * u + 1, row + (long long)h * D + ln.e1);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kRopeStages - 1; ++s) fetch(w.t0 + (long long)s * w.step, s);
  Raw8<T> g0, g1;
  if (gain != nullptr) {
    ldraw(gain + ln.e0, g0);
    ldraw(gain + ln.e1, g1);
  }
  int stage = 0;
  TokenSeq seq;
  for (long long t = w.t0; t < p.tokens; t += w.step) {
    fetch(t + (long long)(kRopeStages - 1) * w.step, stage == 0 ? kRopeStages - 1 : stage - 1);
    const int at = stage;
    stage = stage + 1 == kRopeStages ? 0 : stage + 1;
    const TokenPlace pl = token_place<PAGED>(p, (int)t, seq);
    RopeMap map;
    if (w.kind != 2) {
      float c[8], s[8], ga[8], gz[8];
      ln.turn(p, pl.pos, c, s);
      if (gain != nullptr) {
        unraw(g0, ga);
        unraw(g1, gz);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) ga[i] = gz[i] = 1.0f;
      }
      map.set(c, s, ga, gz, p.interleaved != 0);
    }
    long long hs;
    T* const o = rope_heads<T, D, PAGED>(p, pl, (int)t, w.kind, w.count, w.kind == 0 ? q : w.kind == 1 ? k : v, hs);
    cp_async_wait<kRopeStages - 1>();
    if (!pl.on || o == nullptr) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = w.h0 + u * HPW;
      T* oh = o + h * hs;
      Raw8<T> r0, r1;
      st.read(at, 2 * u, r0);
      st.read(at, 2 * u + 1, r1);
      if (w.kind == 2) {
        if (h < w.count) {
          straw(oh + ln.e0, r0);
          straw(oh + ln.e1, r1);
        }
        continue;
      }
      float a[8], z[8];
      unraw(r0, a);
      unraw(r1, z);
      float inv = 1.0f;
      if (gain != nullptr) inv = rsqrtf(ln.sum(dot8(a, a, z, z)) * (1.0f / D) + p.eps);
      map.apply(a, z, ln.turns, p.interleaved != 0);
      if (h >= w.count) continue;
      if (pl.pos < 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = z[i] = 0.0f;
      } else {
        scale8(a, a, inv);  // the map is linear: 1/r is applied to the result
        scale8(z, z, inv);
      }
      store8(oh + ln.e0, a);
      store8(oh + ln.e1, z);
    }
  }
  cp_async_wait<0>();
}

// Backward; part as in k_qk_norm_rope_bwd_any.  A warp keeps the partial sums of its kind's gain
// gradient for its 16 columns in registers over all its tokens.  32768 tokens, 32 / 8 heads of 128, bf16:
// 216 us with both gain sums, 1.14 GB, 5.3 TB/s; a copy with this access pattern alone 185 us.
template <typename T, int D, int U>
__global__ void __launch_bounds__(256, 2) k_qk_norm_rope_bwd_vec(T* __restrict__ dqkv, float* __restrict__ part,
                                                                 const T* __restrict__ dq, const T* __restrict__ dk,
                                                                 const T* __restrict__ dv, const T* __restrict__ qkv,
                                                                 const T* __restrict__ q_gain,
                                                                 const T* __restrict__ k_gain, const RopeParams p,
                                                                 const RopeBatches nb) {
  constexpr int HPW = 32 / (D / 16);
  extern __shared__ __align__(16) uint8_t rope_smem[];
  __shared__ float red[8][D];
  __shared__ int kinds[8];
  pdl_launch_dependents();
  pdl_wait();
  const RopeLane<D> ln(p.rot);
  const RopeWork<D, U> w(p, nb, ln.sub);
  const RopeStage<T, 4 * U> st(rope_smem, (int)warp_id());
  const T* gain = w.kind == 0 ? q_gain : w.kind == 1 ? k_gain : nullptr;
  const T* dy = w.kind == 0 ? dq : w.kind == 1 ? dk : dv;
  const long long last = w.on && dy != nullptr ? p.tokens : 0;
  auto fetch = [&](long long t, int stage) {
    if (t < last) {
      const int b = (int)((unsigned)t / (unsigned)p.seq), sq = (int)t - b * p.seq;
      const T* y = dy + ((long long)b * w.count * p.seq + sq) * D;
      const T* x = qkv + t * p.ld + (long long)w.col * D;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = w.h0 + u * HPW;
        if (h >= w.count) continue;
        const T* yh = y + (long long)h * p.seq * D;
        st.fetch(stage, 4 * u, yh + ln.e0);
        st.fetch(stage, 4 * u + 1, yh + ln.e1);
        if (gain == nullptr) continue;
        st.fetch(stage, 4 * u + 2, x + (long long)h * D + ln.e0);
        st.fetch(stage, 4 * u + 3, x + (long long)h * D + ln.e1);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int u = 0; u < U; ++u)  // heads that the batch lacks read as zeros
    if (w.h0 + u * HPW >= w.count) st.zero(4 * u, 4);
#pragma unroll
  for (int s = 0; s < kRopeStages - 1; ++s) fetch(w.t0 + (long long)s * w.step, s);
  Raw8<T> g0, g1;
  if (gain != nullptr) {
    ldraw(gain + ln.e0, g0);
    ldraw(gain + ln.e1, g1);
  }
  float acc0[8] = {}, acc1[8] = {};
  int stage = 0;
  TokenSeq seq;
  for (long long t = w.t0; t < last; t += w.step) {
    fetch(t + (long long)(kRopeStages - 1) * w.step, stage == 0 ? kRopeStages - 1 : stage - 1);
    const int at = stage;
    stage = stage + 1 == kRopeStages ? 0 : stage + 1;
    const TokenPlace pl = token_place<false>(p, (int)t, seq);
    float c[8], s[8];
    if (w.kind != 2) ln.turn(p, pl.pos, c, s);
    cp_async_wait<kRopeStages - 1>();
    T* row = dqkv + t * p.ld_out + (long long)w.col * D;
    if (pl.pos < 0 && w.kind != 2) {  // no position: zeros whatever dy and x hold, and nothing for the gains
      const float none[8] = {};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = w.h0 + u * HPW;
        if (h >= w.count) continue;
        store8(row + (long long)h * D + ln.e0, none);
        store8(row + (long long)h * D + ln.e1, none);
      }
      continue;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = w.h0 + u * HPW;
      Raw8<T> r0, r1;
      st.read(at, 4 * u, r0);
      st.read(at, 4 * u + 1, r1);
      if (w.kind == 2) {
        if (h >= w.count) continue;
        straw(row + (long long)h * D + ln.e0, r0);
        straw(row + (long long)h * D + ln.e1, r1);
        continue;
      }
      float a[8], z[8];
      unraw(r0, a);
      unraw(r1, z);
      if (ln.turns) rope_back(a, z, c, s, p.interleaved != 0);
      if (gain != nullptr) {
        float xa[8], xz[8], ga[8], gz[8];
        st.read(at, 4 * u + 2, r0);
        st.read(at, 4 * u + 3, r1);
        unraw(r0, xa);
        unraw(r1, xz);
        unraw(g0, ga);
        unraw(g1, gz);
        float inv = rsqrtf(ln.sum(dot8(xa, xa, xz, xz)) * (1.0f / D) + p.eps);
        if (h >= w.count) inv = 0.0f;  // no head: nothing is added
        scale8(a, a, inv);  // dz / r
        scale8(z, z, inv);
        fma8(acc0, a, xa, acc0);
        fma8(acc1, z, xz, acc1);
        mul8(a, a, ga);  // e / r
        mul8(z, z, gz);
        const float back = ln.sum(dot8(a, xa, z, xz)) * inv * inv * (-1.0f / D);
        fmaw8(a, xa, back, a);  // dx = e / r - x sum(e x / r) / (D r^2)
        fmaw8(z, xz, back, z);
      }
      if (h >= w.count) continue;
      store8(row + (long long)h * D + ln.e0, a);
      store8(row + (long long)h * D + ln.e1, z);
    }
  }
  cp_async_wait<0>();
  if (part == nullptr) return;
  // the warp's heads (lanes of equal l), then the CTA's warps of each kind, in a fixed order
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int o = D / 16; o < 32; o <<= 1) {
      acc0[i] += __shfl_xor_sync(0xffffffffu, acc0[i], o);
      acc1[i] += __shfl_xor_sync(0xffffffffu, acc1[i], o);
    }
    if (ln.sub == 0) {
      red[warp_id()][ln.e0 + i] = acc0[i];
      red[warp_id()][ln.e1 + i] = acc1[i];
    }
  }
  if (lane_id() == 0) kinds[warp_id()] = w.on ? w.kind : 2;
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * D; e += 256) {
    const int kd = e / D, d = e % D;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (kinds[i] == kd) sum += red[i][d];
    part[((long long)blockIdx.x * 2 + kd) * D + d] = sum;
  }
}

// dq_gain (blockIdx.x 0) and dk_gain (1): 32 columns per CTA, the partial rows of the nparts CTAs added
// by eight warps, a contiguous eighth each, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256) k_rope_gain_sum(T* __restrict__ dq_gain, T* __restrict__ dk_gain,
                                                       const float* __restrict__ part, int nparts, int D) {
  __shared__ float red[8][32];
  pdl_launch_dependents();
  pdl_wait();
  T* out = blockIdx.x == 0 ? dq_gain : dk_gain;
  if (out == nullptr) return;
  const int lane = (int)lane_id(), warp = (int)warp_id(), d = (int)blockIdx.y * 32 + lane;
  const int per = (nparts + 7) / 8, i0 = warp * per, i1 = min(nparts, i0 + per);
  float s = 0.0f;
  if (d < D) {
#pragma unroll 8
    for (int i = i0; i < i1; ++i) s += part[((long long)i * 2 + blockIdx.x) * D + d];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && d < D) {
    for (int w = 1; w < 8; ++w) s += red[w][lane];
    stf(out + d, s);
  }
}

// table[t][i] = cos(t theta^(-2i/rot)), table[t][rot/2 + i] = sin of the same angle, in 64 bits:
// a 32-bit angle at position 131072 would be off by up to 0.008.
__global__ void k_rope_table(float* __restrict__ table, long long positions, int rot, double theta) {
  const int half = rot >> 1;
  const long long n = positions * half;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (long long)gridDim.x * blockDim.x) {
    const long long t = e / half;
    const int i = (int)(e - t * half);
    double s, c;
    sincos((double)t * pow(theta, -2.0 * (double)i / (double)rot), &s, &c);
    table[t * rot + i] = (float)c;
    table[t * rot + half + i] = (float)s;
  }
}

}  // namespace beacon
