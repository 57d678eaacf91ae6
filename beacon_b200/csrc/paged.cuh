// paged.cuh -- attention of new tokens over a paged key/value cache: work distribution, the exact
// SIMT kernel, and the kernel that joins split work.
//
// Sequence s brings q_len = cu_q[s+1] - cu_q[s] new tokens and kv = kv_lens[s] cached ones, the new
// ones last.  New token i sits at p = kv - q_len + i and sees keys j <= p (causal) or j < kv:
//   out = softmax(q k^T / sqrt(D)) v, lse = log sum exp; no key visible: out = 0, lse = -inf.
// A row that sees a score of NaN or +inf, or scores of -inf only, has out = NaN and lse = the logarithm of its
// sum (NaN, +inf, -inf).  All of that is read off the row's maximum, which keeps NaN (max_nan); whether a
// row sees a key at all is counted, never read off the maximum.
// For one KV head the rows are (token, query head of the group), token-major: R = q_len * g.
//
// Work: an item is `rpi` consecutive rows of one (sequence, KV head); its length is the time of the
// 128- (or 64-) key tiles its last row sees, at least one, behind `item_cost` for its start and end.
// All items laid end to end (sequence, KV head, item, tile) are cut into gridDim.x equal runs, one per
// CTA, so that one long context fills the GPU as well as many short ones and the SMs finish together; a
// tile is of the run that holds its end.  A run's first and last item may be partial: their unnormalised
// rows (O, m, l) go to two workspace slots of the CTA and are added up in tile order, so results do not
// depend on timing.  Every CTA finds its run itself from cu_q and kv_lens (one warp, 32 sequences per
// step): no plan, no host copy.
#pragma once

#include "rope.cuh"
#include "sm100.cuh"

namespace beacon {

// The split item that begins in a CTA's run, for the join.
struct __align__(16) PagedHead {
  int q0, kvh, row0, rows;  // the sequence's first token, KV head, first row and rows (0: none begins here)
  int pieces;
  int lim;                  // keys that the sequence's first new token sees (causal; may be negative), or all keys
  int pad[2];
};

struct PagedParams {
  PagedSeqs pg;
  int Hq, Hkv, D, g;         // g = Hq / Hkv
  int causal;
  int rpi;                   // rows per item
  int item_cost;             // time of an item's start and end
  int half_rows;             // items of at most so many rows take HW, not W, per tile
  float scale;               // 1 / sqrt(D)
  long long q_stride;        // elements between token rows of q
  long long tokens;
  void* out;                 // [tokens, Hq, D]
  float* lse;                // [tokens, Hq] or null
  PagedHead* heads;          // [gridDim.x] the split item that begins in this CTA's run
  unsigned int* done;        // [gridDim.x, kPagedParts] finished pieces (paged_last_piece)
  float* part_o;             // [slots, D / 4, rpi, 4] (paged_part)
  float2* part_ml;           // [2 * gridDim.x, rpi] (running maximum, in log2 units; sum)
};

enum : unsigned int {
  kSitePagedLens = 0x611,  // cu_q or kv_lens reach past the query rows or the page table
  kSitePagedPage = 0x612,  // a page index outside the cache
  kSitePagedMerge = 0x613,
};

// One contiguous piece of an item: tiles [a, b) of its n.
struct PagedItem {
  int seq, kvh, row0;  // first row within the sequence's R
  int q0, q_len, kv;   // first token, new tokens, cached tokens of the sequence
  int a, b, n;
  int first, pieces;   // run of the item's first piece, and its pieces
};

// Tiles of item i of a sequence.  The walk is 32-bit arithmetic: the host bounds the length of all work below
// 2^31, and the 64-bit divisions cost a decode step more than its loads.
__device__ __forceinline__ int paged_tiles(const PagedParams& p, int i, int q_len, int kv, int kt) {
  int keys = kv;
  if (p.causal) {
    const unsigned rows = min((unsigned)(i + 1) * (unsigned)p.rpi, (unsigned)q_len * (unsigned)p.g);
    keys = max(0, kv - q_len + (int)((rows - 1u) / (unsigned)p.g) + 1);
  }
  return max(1, (int)(((unsigned)keys + (unsigned)kt - 1u) / (unsigned)kt));
}
__device__ __forceinline__ int paged_items(int q_len, int g, int rpi) {
  return (int)(((unsigned)q_len * (unsigned)g + (unsigned)rpi - 1u) / (unsigned)rpi);
}
// First token, new tokens and cached tokens of sequence s, held inside the tensors that they index; whether cu_q
// does not decrease there.
__device__ __forceinline__ bool paged_lens(const PagedParams& p, int s, int& q0, int& q_len, int& kv) {
  q0 = __ldg(p.pg.cu_q + s);
  int q1 = __ldg(p.pg.cu_q + s + 1);
  kv = max(0, __ldg(p.pg.kv_lens + s));
  const bool rises = q1 >= q0;
  const long long most = (long long)p.pg.max_pages * p.pg.page_size;
  if (q0 < 0 || !rises || q1 > p.tokens || kv > most) {
    record_fault(kFaultIndex, kSitePagedLens);
    q0 = min(max(q0, 0), (int)p.tokens);
    q1 = min(max(q1, q0), (int)p.tokens);
    kv = (int)min((long long)kv, most);
  }
  q_len = q1 - q0;
  return rises;
}

// A run, walked item by item by one warp (every lane holds the same state).  KT keys make a tile; W is its
// time, HW that of one of an item of at most half_rows rows.
template <int KT, int W = 1, int HW = 1>
struct PagedWalk {
  int begin, end, chunk;  // the run; its length, that of all runs but the last
  int pos;                // where the next item begins
  int seq, kvh, item;
  int q0, q_len, kv, items;

  __device__ __forceinline__ static int weight(const PagedParams& p, int i, int q_len) {
    if constexpr (W == HW) return W;
    return q_len * p.g - i * p.rpi <= p.half_rows ? HW : W;
  }
  // Of one KV head of sequence s; falls: set where cu_q decreases.
  __device__ __forceinline__ static int work(const PagedParams& p, int s, bool& falls) {
    if (s >= p.pg.seqs) return 0;
    int q0, q_len, kv;
    if (!paged_lens(p, s, q0, q_len, kv)) falls = true;
    const int n = paged_items(q_len, p.g, p.rpi);
    if (n == 0) return 0;
    int w = n * p.item_cost + weight(p, n - 1, q_len) * paged_tiles(p, n - 1, q_len, kv, KT);
    if (!p.causal) return w + (n - 1) * W * paged_tiles(p, 0, q_len, kv, KT);
    for (int i = 0; i < n - 1; ++i) w += W * paged_tiles(p, i, q_len, kv, KT);
    return w;
  }
  // Run `run` of `runs`.
  __device__ __forceinline__ void start(const PagedParams& p, int run, int runs) {
    const int lane = (int)lane_id();
    begin = end = pos = seq = kvh = item = q0 = q_len = kv = items = 0;  // an empty run is never walked
    bool falls = false;
    const int w0 = work(p, lane, falls);
    int total = w0;
#pragma unroll 1
    for (int s = lane + 32; s < p.pg.seqs; s += 32) total += work(p, s, falls);
    // Sequences that overlap may hold more than p.tokens rows together, which the host's bound on the length of
    // all work does not cover: such a call does nothing.
    if (__any_sync(0xffffffffu, falls)) return;
    total = __reduce_add_sync(0xffffffffu, total) * p.Hkv;
    chunk = max(W > HW ? W : HW, (int)(((unsigned)total + (unsigned)runs - 1u) / (unsigned)runs));
    const int from = (int)min((unsigned)run * (unsigned)chunk, (unsigned)total);
    if (from >= total) return;
    int at = from;
#pragma unroll 1
    for (int s0 = 0; s0 < p.pg.seqs; s0 += 32) {
      const int per_head = s0 == 0 ? w0 : work(p, s0 + lane, falls);
      int sum = per_head * p.Hkv;  // inclusive prefix sum
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, at < sum);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        const unsigned head_work = (unsigned)__shfl_sync(0xffffffffu, per_head, l);
        at -= __shfl_sync(0xffffffffu, sum, l) - (int)head_work * p.Hkv;
        seq = s0 + l;
        enter(p);
        kvh = (int)((unsigned)at / head_work);
        at -= kvh * (int)head_work;
#pragma unroll 1
        for (int n; at >= (n = length(p)); ++item) at -= n;
        pos = from - at;
        begin = from;
        end = min(from + chunk, total);
        return;
      }
      at -= __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __device__ __forceinline__ void enter(const PagedParams& p) {
    paged_lens(p, seq, q0, q_len, kv);
    items = paged_items(q_len, p.g, p.rpi);
  }
  __device__ __forceinline__ int length(const PagedParams& p) const {
    return p.item_cost + weight(p, item, q_len) * paged_tiles(p, item, q_len, kv, KT);
  }
  // The next piece; false at the end of the run.
  __device__ __forceinline__ bool next(const PagedParams& p, PagedItem& x) {
#pragma unroll 1
    while (pos < end) {
      const int w = weight(p, item, q_len), at = pos + p.item_cost;
      x.seq = seq;
      x.kvh = kvh;
      x.row0 = item * p.rpi;
      x.q0 = q0;
      x.q_len = q_len;
      x.kv = kv;
      x.n = paged_tiles(p, item, q_len, kv, KT);
      x.a = begin > at ? (begin - at) / w : 0;
      x.b = end > at ? min(x.n, (end - at) / w) : 0;
      x.first = (int)((unsigned)(at + w - 1) / (unsigned)chunk);
      x.pieces = (int)((unsigned)(at + x.n * w - 1) / (unsigned)chunk) - x.first + 1;
      pos = at + x.n * w;
      if (++item >= items) {
        item = 0;
        if (++kvh >= p.Hkv) {
          kvh = 0;
          if (pos < end) {
#pragma unroll 1
            do {
              ++seq;
              enter(p);
            } while (items == 0 && seq + 1 < p.pg.seqs);  // work is left, so a sequence with tokens follows
          }
        }
      }
      if (x.a < x.b) return true;
    }
    return false;
  }
};

__device__ __forceinline__ PagedHead paged_head(const PagedParams& p, const PagedItem& x) {
  return PagedHead{x.q0, x.kvh, x.row0, min(p.rpi, x.q_len * p.g - x.row0), x.pieces, p.causal ? x.kv - x.q_len + 1 : x.kv};
}

// Maxima that keep NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// What a row's sums are multiplied by, and its lse, from its maximum m (log2 units) and sum l of 2^(s - m).
__device__ __forceinline__ float paged_inv(float m, float l) {
  return fabsf(m) < INFINITY ? 1.0f / l : __uint_as_float(0x7fffffffu);
}
__device__ __forceinline__ float paged_lse(float m, float log2_l) {
  return fabsf(m) < INFINITY ? (m + log2_l) * 0.69314718055994531f : m;
}
// Workspace slot of a partial piece: a piece that continues an item is the run's first.
__device__ __forceinline__ int paged_slot(const PagedItem& x) { return 2 * (int)blockIdx.x + (x.a > 0 ? 0 : 1); }

// Columns [4 c, 4 c + 4) of row r of a workspace slot.  Rows lie side by side: the kernels hold a row per
// thread, and 32 of them store or load 512 contiguous bytes (a row-major slot made the end of a split
// piece cost 14 us, mostly in its uncoalesced accesses).
__device__ __forceinline__ float4* paged_part(const PagedParams& p, long long slot, int c, int r) {
  return reinterpret_cast<float4*>(p.part_o) + (slot * (p.D / 4) + c) * p.rpi + r;
}

// The runs that hold pieces of a split item: a run's first piece may continue an item, its last may begin one.
struct PagedPieces {
  int first, n;
  __device__ __forceinline__ long long slot(int i) const { return i == 0 ? 2LL * first + 1 : 2LL * (first + i); }
};
__device__ __forceinline__ PagedPieces paged_pieces(const PagedItem& x) { return PagedPieces{x.first, x.pieces}; }

// Pieces finished per split item (by its first run) and part of its rows.  The counters lie in the call's
// workspace and k_paged_clear, launched ahead on the stream, zeroes them for every execution of the call,
// replays of a captured one included: whatever the workspace held before, and whatever runs beside the
// call with a workspace of its own, no count of another launch is ever seen.  It costs 0.65 us of GPU time
// beside a decode of 10 us, and 2.4 us of the host's.
constexpr int kPagedMaxRuns = 160, kPagedParts = 16;
__global__ void __launch_bounds__(256) k_paged_clear(uint4* __restrict__ done, int n) {
  pdl_launch_dependents();
  pdl_wait();
  for (int i = (int)(blockIdx.x * 256 + threadIdx.x); i < n; i += (int)gridDim.x * 256) done[i] = make_uint4(0u, 0u, 0u, 0u);
}

// One warp, after its part of a piece has been written: whether that part of every piece now has been.  One
// lane's release-acquire add stands for the warp, ordered with the others' accesses by the warp
// barriers around it (a fence in every lane and a relaxed add took twice as long).
__device__ __forceinline__ bool paged_last_piece(const PagedParams& p, const PagedPieces& pc, int part) {
  __syncwarp();
  unsigned int last = 0u;
  if (lane_id() == 0) {
    unsigned int before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                 : "=r"(before)
                 : "l"(p.done + pc.first * kPagedParts + part)
                 : "memory");
    last = before == (unsigned int)pc.n - 1u ? 1u : 0u;
  }
  last = __shfl_sync(0xffffffffu, last, 0);
  __syncwarp();
  return last != 0u;
}

// One warp, before its part of a piece is written: whether that part of every other piece has been.  If so
// this piece's rows need not be written.
__device__ __forceinline__ bool paged_others_done(const PagedParams& p, const PagedPieces& pc, int part) {
  __syncwarp();
  unsigned int all = 0u;
  if (lane_id() == 0) {
    unsigned int n;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(p.done + pc.first * kPagedParts + part) : "memory");
    all = n == (unsigned int)pc.n - 1u ? 1u : 0u;
  }
  all = __shfl_sync(0xffffffffu, all, 0);
  __syncwarp();
  return all != 0u;
}

// Keys that row r (of R) of a piece sees.
__device__ __forceinline__ int paged_limit(const PagedParams& p, const PagedItem& x, int r) {
  return p.causal ? max(0, x.kv - x.q_len + r / p.g + 1) : x.kv;
}

// Element offset of key j of a sequence for a KV head, or -1 when its page is not in the cache.
__device__ __forceinline__ long long paged_key(const PagedSeqs& g, int seq, int kvh, int j) {
  const int pi = j / g.page_size;
  const int page = __ldg(g.page_table + (long long)seq * g.table_stride + pi);
  if (page < 0 || page >= g.num_pages) {
    record_fault(kFaultIndex, kSitePagedPage);
    return -1;
  }
  return (long long)page * g.page_stride + (long long)kvh * g.head_stride +
         (long long)(j - pi * g.page_size) * g.token_stride;
}

// ---------------------------------------------------------------------------
// Exact path: float32 (and bf16 calls that the other kernels' loads cannot serve), fp32 FFMA, expf.
//
// 256 threads; items of 64 rows, tiles of 64 keys; Q, K, V and P in shared memory as fp32.  Thread
// (ty, tx) of 16 x 16 holds rows ty + 16 i: 4 keys of S each and D/16 columns of O; a warp without a row
// of the item skips the arithmetic, so a decode step pays for its few rows only.  K and V of the next
// tile are copied while this one is used (cp.async where rows are 16-byte aligned), its cache offsets
// looked up one tile earlier still.  Bound: FFMA and shared-memory loads for full items (two 16-byte
// loads per 16 FMA), the serial phases of a run for short ones.
// ---------------------------------------------------------------------------
constexpr int kPagedSimtKt = 64, kPagedSimtRows = 64;
template <int D>
constexpr size_t paged_simt_smem() {
  return sizeof(float) * ((size_t)(kPagedSimtRows + 4 * kPagedSimtKt) * (D + 4) +
                          (size_t)kPagedSimtRows * (kPagedSimtKt + 4) + 2 * kPagedSimtRows) +
         sizeof(long long) * 2 * kPagedSimtKt;
}

// Exact form: products and sums in fp32 FFMA, 64 rows x 64 keys per step, 4 x 4 scores per thread, keys and
// values copied a tile ahead.  Bound: FFMA issue for long work.  For short work (8 sequences of 33-1500
// keys, 1-40 new tokens, 8 / 4 heads of 64: 27 us) a run is one 64-key step, 2-3 us of FFMA; the rest is what
// stands before and after it: finding the run, page lookups, copies, partial rows, the join's launch.  Also takes bf16 calls that
// neither other kernel can: head_dim 16 and 32, and rows that are not 16-byte aligned.
// ASYNC: T is float and the caches' rows are 16-byte aligned.
template <typename T, int D, bool ASYNC>
__global__ void __launch_bounds__(256) k_paged_attn_simt(const T* __restrict__ q, const T* __restrict__ kc,
                                                         const T* __restrict__ vc, const PagedParams p) {
  constexpr int KT = kPagedSimtKt, BM = kPagedSimtRows, LD = D + 4, LP = KT + 4, RT = BM / 16, CT = D / 16;
  constexpr int CV = CT < 4 ? CT : 4;  // columns per load: tx * CV + 16 CV g + e
  extern __shared__ __align__(16) float fsm[];
  float* sq = fsm;
  float* sk = sq + BM * LD;             // [2][KT]
  float* sv = sk + 2 * KT * LD;         // [2][KT]
  float* sp = sv + 2 * KT * LD;
  float* s_m = sp + BM * LP;
  float* s_l = s_m + BM;
  long long* s_off = reinterpret_cast<long long*>(s_l + BM);  // [2][KT] cache offsets of a tile's keys, -1: none
  __shared__ PagedItem item;
  __shared__ int more;
  const int tid = (int)threadIdx.x;
  const int ty = tid >> 4, tx = tid & 15;
  pdl_launch_dependents();
  pdl_wait();
  PagedWalk<KT> walk;
  if (warp_id() == 0) {
    walk.start(p, (int)blockIdx.x, (int)gridDim.x);
    if (tid == 0) p.heads[blockIdx.x] = PagedHead{};
  }
  const int group = p.g;
  for (;;) {
    __syncthreads();
    if (warp_id() == 0) {
      PagedItem x;
      const bool ok = walk.next(p, x);
      if (tid == 0) {
        more = ok ? 1 : 0;
        item = x;
        if (ok && x.a == 0 && x.b < x.n) p.heads[blockIdx.x] = paged_head(p, x);
      }
    }
    __syncthreads();
    if (!more) break;
    const PagedItem x = item;
    const int rows = min(p.rpi, x.q_len * group - x.row0);
    const bool works = (ty & ~1) < rows;  // the warp has a row
    auto lookup = [&](int j) -> long long {  // cache offset of key tid of a tile
      const int key = j * KT + tid;
      return tid < KT && j < x.b && key < x.kv ? paged_key(p.pg, x.seq, x.kvh, key) : -1;
    };
    auto copy = [&](int buf) {
      for (int e = tid; e < KT * (D / 4); e += 256) {
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        const long long at = s_off[buf * KT + r];
        float* dk = sk + (buf * KT + r) * LD + d;
        float* dv = sv + (buf * KT + r) * LD + d;
        if constexpr (ASYNC) {
          const bool have = at >= 0;
          cp_async16_or_zero(smem_u32(dk), kc + (have ? at + d : 0), have);
          cp_async16_or_zero(smem_u32(dv), vc + (have ? at + d : 0), have);
        } else {
          float4 kf = make_float4(0.f, 0.f, 0.f, 0.f), vf = kf;
          if (at >= 0) {
            const T *ks = kc + at + d, *vs = vc + at + d;
            kf = make_float4(ldf(ks), ldf(ks + 1), ldf(ks + 2), ldf(ks + 3));
            vf = make_float4(ldf(vs), ldf(vs + 1), ldf(vs + 2), ldf(vs + 3));
          }
          *reinterpret_cast<float4*>(dk) = kf;
          *reinterpret_cast<float4*>(dv) = vf;
        }
      }
      cp_async_commit();
    };
    const long long off0 = lookup(x.a);
    long long off = lookup(x.a + 1);  // of the tile after the one that is copied next
    if (tid < KT) s_off[tid] = off0;
    __syncthreads();
    copy(0);
    {  // query rows, four threads each
      const int r = tid >> 2, fr = x.row0 + r;
      const T* src = q + (long long)(x.q0 + fr / group) * p.q_stride + ((long long)x.kvh * group + fr % group) * D;
      if (r < ((rows + 15) & ~15)) {
#pragma unroll 8
        for (int d = tid & 3; d < D; d += 4) sq[r * LD + d] = r < rows ? ldf(src + d) * p.scale : 0.0f;
      }
    }
    if (tid < BM) {
      s_m[tid] = -INFINITY;
      s_l[tid] = 0.0f;
    }
    float o[RT][CT] = {};
    for (int j = x.a; j < x.b; ++j) {
      const int k0 = j * KT, buf = (j - x.a) & 1;
      if (j + 1 < x.b) {
        if (tid < KT) s_off[(buf ^ 1) * KT + tid] = off;
        __syncthreads();  // the next tile's offsets are there, and its buffer has been used
        copy(buf ^ 1);
        off = lookup(j + 2);
        cp_async_wait<1>();
      } else {
        cp_async_wait<0>();
      }
      __syncthreads();
      if (!works) continue;
      const float* kt = sk + buf * KT * LD;
      const float* vt = sv + buf * KT * LD;
      float s[RT][4] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 kf[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) kf[c] = *reinterpret_cast<const float4*>(kt + (tx + 16 * c) * LD + d);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (i > 0 && 16 * i >= rows) break;
          const float4 qf = *reinterpret_cast<const float4*>(sq + (ty + 16 * i) * LD + d);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            s[i][c] = fmaf(qf.x, kf[c].x, fmaf(qf.y, kf[c].y, fmaf(qf.z, kf[c].z, fmaf(qf.w, kf[c].w, s[i][c]))));
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (i > 0 && 16 * i >= rows) break;
        const int r = ty + 16 * i;
        const int limit = (r < rows ? paged_limit(p, x, x.row0 + r) : 0) - k0;
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (tx + 16 * c >= limit) s[i][c] = -INFINITY;
          mx = max_nan(mx, s[i][c]);
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const float m_old = s_m[r], m_new = max_nan(m_old, mx);
        const float base = m_new == -INFINITY ? 0.0f : m_new;  // a row that has seen no key yet
        float sum = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float e = expf(s[i][c] - base);
          sp[r * LP + tx + 16 * c] = e;
          sum += e;
        }
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const float alpha = expf(m_old - base);
        __syncwarp();
        if (tx == 0) {
          s_m[r] = m_new;
          s_l[r] = s_l[r] * alpha + sum;
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) o[i][c] *= alpha;
      }
      __syncwarp();  // a row's probabilities are written and read by one warp
#pragma unroll 4
      for (int kk = 0; kk < KT; kk += 4) {
        float vf[4][CT];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int c = 0; c < CT; c += CV) {
            const float* src = vt + (kk + e) * LD + tx * CV + 16 * c;
            if constexpr (CV == 4) *reinterpret_cast<float4*>(&vf[e][c]) = *reinterpret_cast<const float4*>(src);
            else if constexpr (CV == 2) *reinterpret_cast<float2*>(&vf[e][c]) = *reinterpret_cast<const float2*>(src);
            else vf[e][c] = *src;
          }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (i > 0 && 16 * i >= rows) break;
          const float4 pf = *reinterpret_cast<const float4*>(sp + (ty + 16 * i) * LP + kk);
#pragma unroll
          for (int c = 0; c < CT; ++c)
            o[i][c] = fmaf(pf.w, vf[3][c], fmaf(pf.z, vf[2][c], fmaf(pf.y, vf[1][c], fmaf(pf.x, vf[0][c], o[i][c]))));
        }
      }
    }
    __syncwarp();
    const bool whole = x.a == 0 && x.b == x.n;
    const int slot = paged_slot(x);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty + 16 * i;
      if (r >= rows) continue;
      const float m = s_m[r], l = s_l[r];
      const int fr = x.row0 + r;
      const long long at = (long long)(x.q0 + fr / group) * p.Hq + (long long)x.kvh * group + fr % group;
      const bool sees = paged_limit(p, x, fr) > 0;
      const float inv = paged_inv(m, l);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const int d = tx * CV + 16 * (c - c % CV) + c % CV;
        if (whole) stf((T*)p.out + at * D + d, sees ? o[i][c] * inv : 0.0f);
        else reinterpret_cast<float*>(paged_part(p, slot, d / 4, r))[d % 4] = o[i][c];
      }
      if (tx != 0) continue;
      if (!whole) p.part_ml[(long long)slot * p.rpi + r] = make_float2(m * 1.4426950408889634f, l);
      else if (p.lse != nullptr) p.lse[at] = fabsf(m) < INFINITY ? m + logf(l) : m;
    }
  }
}

// Joins the split items that p.heads lists: their blocks of 32 rows x 16 columns are dealt out to the
// grid's warps, a row per lane.  The item that begins in run c has its first piece in slot 2c + 1 and
// the others in slots 2(c + 1), 2(c + 2), .. in order.  With M = max m:
// out = sum 2^(m - M) O / sum 2^(m - M) l.  Bound: latency (its pieces are read side by side): 5.4 us alone
// after 2048 new tokens over 32768 keys; launched ahead, it starts as the attention kernel ends.
constexpr int kPagedMostRuns = 320;  // of any attention kernel that leaves its joins to this one
template <typename T>
__global__ void __launch_bounds__(256) k_paged_join(const PagedParams p, int runs) {
  __shared__ PagedHead heads[kPagedMostRuns];
  __shared__ int first[kPagedMostRuns + 1];  // 32-row blocks of the items before
  pdl_launch_dependents();
  pdl_wait();
  const int lane = (int)lane_id();
  for (int c = (int)threadIdx.x; c < runs; c += 256) heads[c] = p.heads[c];
  __syncthreads();
  if (warp_id() == 0) {
    int sum = 0;
    for (int c0 = 0; c0 < runs; c0 += 32) {
      const int blocks = c0 + lane < runs ? (heads[c0 + lane].rows + 31) / 32 : 0;
      int end = blocks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      if (c0 + lane < runs) first[c0 + lane] = sum + end - blocks;
      sum += __shfl_sync(0xffffffffu, end, 31);
    }
    if (lane == 0) first[runs] = sum;
  }
  __syncthreads();
  const int parts = p.D / 16, total = first[runs] * parts;
  for (int k = (int)(blockIdx.x * 8 + warp_id()); k < total; k += (int)gridDim.x * 8) {
    const int block = k / parts, c0 = (k - block * parts) * 4;
    int c = 0;
    for (int step = 256; step > 0; step >>= 1)
      if (c + step < runs && first[c + step] <= block) c += step;  // the last item that starts at or before it
    const PagedHead h = heads[c];
    const int r = (block - first[c]) * 32 + lane;
    const PagedPieces pc{c, h.pieces};
    if (r >= h.rows) continue;
    // one pass over the pieces with a running maximum, four pieces' loads at a time.  A piece without a
    // key of this row has left old values in its slot: read all the same, so that no load waits for
    // another, and passed over.
    float mx = -INFINITY, l = 0.0f, o[16] = {};
    for (int i0 = 0; i0 < pc.n; i0 += 4) {
      float2 ml[4];
      float4 v[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long slot = pc.slot(min(i0 + i, pc.n - 1));
        ml[i] = p.part_ml[slot * p.rpi + r];
        if (i0 + i >= pc.n) ml[i].x = -INFINITY;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[i][q] = *paged_part(p, slot, c0 + q, r);
      }
      const float m_new = max3_nan(max_nan(ml[0].x, ml[1].x), max_nan(ml[2].x, ml[3].x), mx);
      if (m_new == -INFINITY) continue;
      const float alpha = exp2f(mx - m_new);
      mx = m_new;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] *= alpha;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (ml[i].x == -INFINITY) continue;
        const float wgt = exp2f(ml[i].x - mx);
        l = fmaf(ml[i].y, wgt, l);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          o[4 * q] = fmaf(v[i][q].x, wgt, o[4 * q]);
          o[4 * q + 1] = fmaf(v[i][q].y, wgt, o[4 * q + 1]);
          o[4 * q + 2] = fmaf(v[i][q].z, wgt, o[4 * q + 2]);
          o[4 * q + 3] = fmaf(v[i][q].w, wgt, o[4 * q + 3]);
        }
      }
    }
    const int fr = h.row0 + r;
    const long long at = (long long)(h.q0 + fr / p.g) * p.Hq + (long long)h.kvh * p.g + fr % p.g;
    const bool sees = (p.causal ? h.lim + fr / p.g : h.lim) > 0;
    const float inv = paged_inv(mx, l);
    T* dst = (T*)p.out + at * p.D + 4 * c0;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = sees ? o[e] * inv : 0.0f;
    if ((reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
      store8(dst, *reinterpret_cast<const float(*)[8]>(&o[0]));
      store8(dst + 8, *reinterpret_cast<const float(*)[8]>(&o[8]));
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) stf(dst + e, o[e]);
    }
    if (c0 == 0 && p.lse != nullptr) p.lse[at] = paged_lse(mx, log2f(l));
  }
}

}  // namespace beacon
