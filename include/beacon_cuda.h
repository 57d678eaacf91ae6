/*
 * beacon_cuda.h -- C ABI of libbeacon_cuda.so, the B200 (sm_100a) kernels behind
 * beacon's launcher traits.
 *
 * One entry point per kernel ID of crates/beacon-cuda (the IDs equal the
 * launcher strings of crates/beacon-adjoint-table/src/lib.rs:53-116).  Each takes
 * plain device pointers, explicit shapes, a dtype and a CUDA stream, because the
 * reference's typed traits drop the shapes before KernelLauncher::launch
 * (e.g. `let _ = (m, k, n)` at crates/beacon-cuda/src/matmul.rs:27).
 *
 * Conventions
 *  - Row-major contiguous tensors: matrices [rows, cols]; attention tensors
 *    [B, H, S, D]; LSE [B, H, S] float32; RMSNorm statistic rms and LayerNorm
 *    statistics mean, invstd: [tokens] float32.
 *  - `dtype` is a beacon_dtype (crates/beacon-core/src/dtype.rs:1-6 order).
 *    BEACON_BF16: bf16 operands, fp32 accumulation on tcgen05 tensor cores.
 *    BEACON_F32 : exact fp32 FFMA (no TF32) -- the 1e-5 parity path.
 *  - `stream` is a cudaStream_t (NULL = legacy default stream).  Every call is
 *    asynchronous on that stream and never synchronises the device, except
 *    where a comment says it may grow the library's internal workspace.
 *  - Concurrency: calls on different streams may overlap on the GPU, except that
 *    calls which take their scratch from the library's per-device workspace
 *    (workspace = NULL) share that one buffer: give each stream its own workspace
 *    when such calls may overlap.  The persistent kernels (attention forward, dK/dV, dQ)
 *    take their work items from one of 64 counter slots per device, rotating
 *    launch by launch and reset by each launch's last CTA: up to 64 such
 *    launches may be in flight on one device at once.  A captured launch keeps the
 *    slot of its capture: replay it only while none of these kernels that another
 *    stream launched is in flight.  Paged attention counts in its workspace
 *    and has no such limit.
 *  - Return value: a beacon_status that maps 1:1 onto beacon-cuda's LaunchError
 *    variants (crates/beacon-cuda/src/error.rs:4-13); 0 is Ok.  The message of
 *    the last error on the calling thread is available from beacon_last_error().
 *  - No entry point falls back to the CPU.  A device without sm_100 support
 *    fails with BEACON_ERR_MODULE_LOAD.
 */
#ifndef BEACON_CUDA_H
#define BEACON_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* LaunchError variants, crates/beacon-cuda/src/error.rs:4-13 */
typedef enum beacon_status {
    BEACON_OK = 0,
    BEACON_ERR_UNIMPLEMENTED = 1,
    BEACON_ERR_INVALID_LAUNCH_CONFIG = 2,
    BEACON_ERR_MODULE_LOAD = 3,
    BEACON_ERR_FUNCTION_NOT_FOUND = 4,
    BEACON_ERR_CUDA = 5,
    BEACON_ERR_CUBLAS = 6,
    BEACON_ERR_OUT_OF_MEMORY = 7,
    BEACON_ERR_SHAPE_MISMATCH = 8
} beacon_status;

/* DType, crates/beacon-core/src/dtype.rs:1-7 */
typedef enum beacon_dtype {
    BEACON_F32 = 0,
    BEACON_F16 = 1,
    BEACON_BF16 = 2,
    BEACON_FP8E4M3 = 3
} beacon_dtype;

/* CastKind, crates/beacon-cuda/src/elementwise.rs:27-44 */
typedef enum beacon_cast_kind {
    BEACON_CAST_F32_TO_FP8E4M3 = 0,
    BEACON_CAST_FP8E4M3_TO_F32 = 1,
    BEACON_CAST_F32_TO_BF16 = 2,
    BEACON_CAST_BF16_TO_F32 = 3
} beacon_cast_kind;

/* ---- library / errors ----------------------------------------------------- */

/* Library ABI version (major * 10000 + minor * 100 + patch). */
int beacon_version(void);

/* Copies the calling thread's last error message into buf (NUL-terminated,
 * truncated to len) and returns the status that produced it. */
int beacon_last_error(char* buf, size_t len);

/* Reads and clears the device-side fault words of `device`:
 * out[0] fault code (0 none, 1 a bounded wait timed out), out[1] site,
 * out[2] number of faults since the last read.  Synchronises the device.
 * Replaces the kernel-completion check of crates/beacon-cuda/src/device.rs:72-74. */
int beacon_device_status(int device, unsigned int out[3]);

/* Number of kernels launched by this library since load (all devices, all threads). */
uint64_t beacon_launch_count(void);

/* Self-checks of device building blocks (no reference counterpart).
 * beacon_diag_wait_timeout: one warp on the current device waits on an mbarrier that
 * nothing completes, with the bounded wait every kernel uses but a limit of `limit_ns`
 * (at most 1 s); the wait gives up, records fault code 1 at site 0x501 (read it with
 * beacon_device_status), the bulk copy the kernel has in flight lands, its TMEM is freed
 * and it returns.  out: 3 device words = {gave up (1), first word of the copy (1),
 * TMEM released (1)}.
 * beacon_diag_exp2_poly: out[i] = 2^in[i] by the FMA-pipe polynomial the attention
 * softmax uses for part of its exponentials (n even); its stated bound is a relative
 * error below 7.5e-5 on [-125.5, 8] and an absolute error below 2^-125 beneath it. */
int beacon_diag_wait_timeout(uint64_t limit_ns, unsigned int* out, void* stream);
int beacon_diag_exp2_poly(float* out, const float* in, int64_t n, void* stream);

/* Device timing of the tensor-core kernels (k_gemm_bf16_tc, k_attn_fwd_tc,
 * k_attn_bwd_dkdv, k_attn_bwd_dq, k_paged_attn_tc, k_paged_attn_dec): while enabled, each launch is bracketed by CUDA events on its
 * own stream.  beacon_profile_read(name, ...) waits for those events and returns the
 * accumulated milliseconds and launch count for `name`; name == NULL resets.
 * No reference counterpart (the reference bench is a stub,
 * crates/beacon-bench/src/main.rs:1-3). */
void beacon_profile_enable(int on);
int beacon_profile_read(const char* kernel, double* total_ms, uint64_t* count);

/* ---- matmul / linear: crates/beacon-cuda/src/matmul.rs ---------------------- */

/* The tile shape the bf16 GEMM entry points choose for an [m, k] x [k, n] product with
 * 16-byte aligned rows on the current device: out[0] rows per tile (128, or 256 for an SM
 * pair), out[1] columns per tile, out[2] tiles, out[3] SMs per tile (1 or 2), out[4] the
 * device's SM count.  No counterpart in the reference: a planning query for launch
 * configuration and benchmarks (wave efficiency = tiles / (ceil(tiles / slots) x slots),
 * slots = SMs / SMs per tile). */
int beacon_matmul_plan(int64_t m, int64_t k, int64_t n, int32_t* out);

/* matmul_fwd (matmul.rs:18-29): out[m,n] = lhs[m,k] . rhs[k,n] */
int beacon_matmul_fwd(void* out, const void* lhs, const void* rhs, int64_t m, int64_t k, int64_t n,
                      int dtype, void* stream);

/* matmul_bwd (matmul.rs:31-44): dlhs[m,k] = dout . rhs^T ; drhs[k,n] = lhs^T . dout.
 * Either gradient pointer may be NULL to skip it. */
int beacon_matmul_bwd(void* dlhs, void* drhs, const void* dout, const void* lhs, const void* rhs,
                      int64_t m, int64_t k, int64_t n, int dtype, void* stream);

/* linear_fwd (matmul.rs:46-58): out[m,n] = x[m,k] . weight[k,n] + bias[n] (bias may be NULL). */
int beacon_linear_fwd(void* out, const void* x, const void* weight, const void* bias, int64_t m, int64_t k,
                      int64_t n, int dtype, void* stream);

/* fp8 e4m3 weights (DType::Fp8E4M3, crates/beacon-core/src/dtype.rs:6; codec dtype.rs:134-195;
 * the reference's "cublasLt fp8" / "fp32 master -> fp8 weights" plan, crates/beacon-cuda/Cargo.toml:7,
 * crates/beacon-train/Cargo.toml:7).  `dtype = BEACON_FP8E4M3` in beacon_matmul_fwd /
 * beacon_linear_fwd means: lhs / x, bias and out are bf16, rhs / weight is fp8 e4m3 [k, n]
 * with scale 1.  The _fp8w_ entry points take the per-tensor dequantisation scale:
 * out = (lhs . decode(rhs)) * scale (+ bias).  The weights are decoded to bf16 (exactly)
 * inside the GEMM pipeline -- TMA brings the fp8 bytes into shared memory, converter warps
 * decode them into the tensor core's operand layout -- so each weight byte is read from
 * HBM once; the scale is applied in the epilogue.  (lhs 16-byte aligned with k % 8 == 0,
 * weights 16-byte aligned with n % 16 == 0; other shapes decode to a bf16 copy in the
 * library workspace first.) */
int beacon_matmul_fp8w_fwd(void* out, const void* lhs, const void* rhs_fp8, float rhs_scale, int64_t m, int64_t k,
                           int64_t n, void* stream);
int beacon_linear_fp8w_fwd(void* out, const void* x, const void* weight_fp8, float weight_scale, const void* bias,
                           int64_t m, int64_t k, int64_t n, void* stream);
/* The same with the scale read from device memory (as beacon_quantize_fp8e4m3 writes it),
 * so no host round trip sits between quantising and using the weights; bias may be NULL. */
int beacon_linear_fp8w_fwd_devscale(void* out, const void* x, const void* weight_fp8, const float* weight_scale_dev,
                                    const void* bias, int64_t m, int64_t k, int64_t n, void* stream);

/* fp32 master -> fp8 e4m3 weights, one scale per tensor (the reference's "fp32 master ->
 * fp8 weights", crates/beacon-train/Cargo.toml:7; no scale convention is fixed there):
 *   amax = max |src| (NaN ignored), scale = amax / 448 (1 when amax is 0),
 *   out[i] = F8E4M3::from_f32(src[i] * (448 / amax))  (crates/beacon-core/src/dtype.rs:163-195,
 *   bit-exact, float32 arithmetic), so src ~ decode(out) * scale.
 * amax and scale are single floats in device memory (written on the stream). */
int beacon_quantize_fp8e4m3(void* out_fp8, float* scale, float* amax, const float* src, int64_t n, void* stream);

/* linear_bwd (matmul.rs:60-78): dx = dout . weight^T ; dweight = x^T . dout ; dbias = sum_rows dout.
 * Any gradient pointer may be NULL to skip it. */
int beacon_linear_bwd(void* dx, void* dweight, void* dbias, const void* dout, const void* x, const void* weight,
                      int64_t m, int64_t k, int64_t n, int dtype, void* stream);

/* ---- attention: crates/beacon-cuda/src/attention.rs ------------------------ */

/* attention_fwd (attention.rs:21-40), kernel `attention_adjoint_fwd`:
 * out = softmax(Q K^T / sqrt(head_dim) + causal mask) V, lse = natural-log logsumexp
 * per query row (float32).  q, k, v, out: [batch, heads, seqlen, head_dim]. */
int beacon_attention_adjoint_fwd(void* out, const void* q, const void* k, const void* v, float* lse,
                                 int64_t batch, int64_t heads, int64_t seqlen, int64_t head_dim, int causal,
                                 int dtype, void* stream);

/* attention_bwd (attention.rs:42-64), kernel `attention_adjoint_bwd`; adjoint entry
 * crates/beacon-adjoint-table/src/lib.rs:86-99 (saved q, k, v, lse; scores recomputed).
 * The forward output is not an argument: the forward kernel runs again, given the saved
 * lse, and forms rowsum(dO * O) from O in tensor memory (O is not written).  Scratch
 * (two fp32 values per query row): `workspace` of at least
 * beacon_attention_bwd_workspace_size(...) bytes, or NULL to use the library's
 * per-device workspace (grown with cudaMalloc on first use; the growth synchronises
 * the device). */
int beacon_attention_adjoint_bwd(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                                 const void* v, const float* lse, int64_t batch, int64_t heads, int64_t seqlen,
                                 int64_t head_dim, int causal, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream);

size_t beacon_attention_bwd_workspace_size(int64_t batch, int64_t q_heads, int64_t seqlen, int64_t head_dim,
                                           int dtype);

/* Grouped-query variants.  No reference counterpart: attention.rs:28-31 has only
 * `heads`; these add kv_heads (q_heads % kv_heads == 0; query head h reads KV head
 * h / (q_heads / kv_heads)).  kv_heads == q_heads is exactly the entry points above.
 * k, v, dk, dv: [batch, kv_heads, seqlen, head_dim]. */
int beacon_attention_gqa_fwd(void* out, const void* q, const void* k, const void* v, float* lse, int64_t batch,
                             int64_t q_heads, int64_t kv_heads, int64_t seqlen, int64_t head_dim, int causal,
                             int dtype, void* stream);
int beacon_attention_gqa_bwd(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                             const void* v, const float* lse, int64_t batch, int64_t q_heads, int64_t kv_heads,
                             int64_t seqlen, int64_t head_dim, int causal, int dtype, void* workspace,
                             size_t workspace_bytes, void* stream);

/* Backward that is also given the forward output `out`, so it skips the
 * recompute; for callers that keep O resident.  No reference counterpart. */
int beacon_attention_bwd_with_out(void* dq, void* dk, void* dv, const void* dout, const void* q, const void* k,
                                  const void* v, const void* out, const float* lse, int64_t batch,
                                  int64_t q_heads, int64_t kv_heads, int64_t seqlen, int64_t head_dim,
                                  int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* ---- RMSNorm: crates/beacon-cuda/src/norm.rs:19-51 -------------------------- */

/* rmsnorm_fwd (norm.rs:20-31): rms[t] = sqrt(mean(x[t]^2) + eps) (float32),
 * out = x * weight / rms.  The reference signature has no eps; its callers pass 1e-5. */
int beacon_rmsnorm_adjoint_fwd(void* out, const void* x, const void* weight, float* rms, int64_t tokens,
                               int64_t dim, float eps, int dtype, void* stream);

/* rmsnorm_bwd (norm.rs:33-50): dx = (w dy)/rms - x sum(w dy x)/(dim rms^3);
 * dweight = sum_t dy x / rms (NULL to skip).  Workspace as for attention. */
int beacon_rmsnorm_adjoint_bwd(void* dx, void* dweight, const void* dy, const void* x, const float* rms,
                               const void* weight, int64_t tokens, int64_t dim, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream);

/* RMSNorm backward that allocates nothing.  No counterpart in the reference: it is
 * for callers that cannot allocate device memory themselves (a launcher that only
 * hands out pointers into one preallocated arena, a path that cannot afford the
 * first-call cudaMalloc and device synchronisation of the library's own workspace).
 * Same arithmetic as beacon_rmsnorm_adjoint_bwd (results agree up to the float32
 * summation order of dweight); the dweight partial sums live in a
 * fixed 4 MiB (1,048,576-float) array compiled into the library, which every GPU
 * that loads the library holds until exit.  dim above 1,048,576 is rejected with
 * BEACON_ERR_INVALID_LAUNCH_CONFIG.  The array's address is looked up on the first
 * call made on each device (make that call before any stream capture).  With CUDA's
 * lazy module loading (the default), the first call into this library on a device --
 * whichever entry point it is -- loads the library's module there, which places the
 * array and may synchronise; make one such call outside any latency-critical region,
 * or load eagerly with CUDA_MODULE_LOADING=EAGER.  All calls share the array: calls
 * that overlap on the GPU race and must be serialised. */
int beacon_rmsnorm_adjoint_bwd_noalloc(void* dx, void* dweight, const void* dy, const void* x, const float* rms,
                                       const void* weight, int64_t tokens, int64_t dim, int dtype, void* stream);

/* RMSNorm fused into the linear layer that consumes it: rmsnorm_fwd (norm.rs:20-31)
 * followed by linear_fwd (matmul.rs:46-58) as
 *     rmsnorm(x, g) . W + b = diag(1 / rms) . x . (diag(g) . W) + b.
 * beacon_rmsnorm_fold_weight writes w_out[i, j] = g[i] * w[i, j] (rounded to dtype), once
 * per weight version.  beacon_rmsnorm_linear_fwd then reads x once for its row statistic
 * rms[t] = sqrt(mean(x[t]^2) + eps) (written: the value rmsnorm_fwd saves for the
 * backward) and runs the GEMM on raw x and the folded weight with 1 / rms[t] applied to
 * each accumulator row in the epilogue (+ bias, may be NULL): no normalised copy of x is
 * written or read.  x [m, k], w_folded [k, n], out [m, n]; f32 or bf16.
 * No reference counterpart as one call (the reference has the two operators). */
int beacon_rmsnorm_fold_weight(void* w_out, const void* gain, const void* w, int64_t k, int64_t n, int dtype,
                               void* stream);
int beacon_rmsnorm_linear_fwd(void* out, float* rms, const void* x, const void* w_folded, const void* bias,
                              int64_t m, int64_t k, int64_t n, float eps, int dtype, void* stream);

/* ---- LayerNorm: crates/beacon-cuda/src/norm.rs:55-95 ----------------------- */

/* layernorm_fwd (norm.rs:56-73): mean[t] = mean_d x[t, d],
 * invstd[t] = 1 / sqrt(mean_d (x[t, d] - mean[t])^2 + eps) (biased variance; both float32),
 * out = (x - mean) * invstd * weight + bias.  The reference signature has no eps; 1e-5 is
 * the convention of the RMSNorm above.  The saved statistics are mean and invstd
 * (adjoint crates/beacon-adjoint-table/src/lib.rs:78-85). */
int beacon_layernorm_adjoint_fwd(void* out, const void* x, const void* weight, const void* bias, float* mean,
                                 float* invstd, int64_t tokens, int64_t dim, float eps, int dtype, void* stream);

/* layernorm_bwd (norm.rs:75-94): with xh = (x - mean) invstd and e = weight dy,
 * dx = invstd (e - mean_d e - xh mean_d(e xh)); dweight = sum_t dy xh; dbias = sum_t dy
 * (either may be NULL).  Workspace as for attention: 4 * min(tokens, 4 * SMs) * dim bytes
 * for each of dweight and dbias requested. */
int beacon_layernorm_adjoint_bwd(void* dx, void* dweight, void* dbias, const void* dy, const void* x,
                                 const float* mean, const float* invstd, const void* weight, int64_t tokens,
                                 int64_t dim, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/* ---- SwiGLU MLP: crates/beacon-cuda/src/mlp.rs:12-52 ----------------------- */

/* swiglu_fwd (mlp.rs:12-29): out[t, dm] = (silu(x Wg) * (x Wu)) Wd;
 * gate_proj, up_proj: [d_model, d_ff]; down_proj: [d_ff, d_model].
 * The gate and up GEMMs run as one tcgen05 GEMM with a SwiGLU epilogue. */
int beacon_swiglu_adjoint_fwd(void* out, const void* x, const void* gate_proj, const void* up_proj,
                              const void* down_proj, int64_t tokens, int64_t d_model, int64_t d_ff, int dtype,
                              void* workspace, size_t workspace_bytes, void* stream);

/* swiglu_bwd (mlp.rs:31-52); adjoint lib.rs:100-107 recomputes gate and up. */
int beacon_swiglu_adjoint_bwd(void* dx, void* dgate_proj, void* dup_proj, void* ddown_proj, const void* dy,
                              const void* x, const void* gate_proj, const void* up_proj, const void* down_proj,
                              int64_t tokens, int64_t d_model, int64_t d_ff, int dtype, void* workspace,
                              size_t workspace_bytes, void* stream);

size_t beacon_swiglu_workspace_size(int64_t tokens, int64_t d_model, int64_t d_ff, int dtype, int backward);

/* ---- pre-norm Llama-style block forward (no reference counterpart) ---------
 * The composition beacon-nn would make of rmsnorm_fwd (norm.rs:19-31), linear_fwd
 * (matmul.rs:46-58), attention_fwd (attention.rs:21-40), residual_add
 * (elementwise.rs:47-55) and swiglu_fwd (mlp.rs:12-29), in seven launches:
 *   h   = x + attention(rmsnorm(x, attn_norm) . w_qkv) . w_o        (causal)
 *   out = h + (silu(xn . w_gate) * (xn . w_up)) . w_down,  xn = rmsnorm(h, ffn_norm)
 * The QKV GEMM stores q, k, v head-major straight from its epilogue, attention writes
 * its output token-major, and both residual adds are GEMM epilogues.
 * x, out: [batch*seq, d_model]; attn_norm, ffn_norm: [d_model];
 * w_qkv: [d_model, (heads + 2*kv_heads)*head_dim] (query heads, then key heads, then
 * value heads); w_o: [heads*head_dim, d_model]; w_gate, w_up: [d_model, d_ff];
 * w_down: [d_ff, d_model].  bf16 only; head_dim 64 or 128; d_model and d_ff multiples
 * of 8; pointers 16-byte aligned.  Scratch (beacon_llama_block_workspace_size bytes,
 * or the library's workspace when `workspace` is NULL) holds, at the offsets the
 * layout in abi_block.inc gives, the normalised rows, both rms vectors, q, k, v, the
 * attention output, h and the SwiGLU activations. */
int beacon_llama_block_fwd(void* out, const void* x, const void* attn_norm, const void* w_qkv, const void* w_o,
                           const void* ffn_norm, const void* w_gate, const void* w_up, const void* w_down,
                           int64_t batch, int64_t seq, int64_t d_model, int64_t heads, int64_t kv_heads,
                           int64_t head_dim, int64_t d_ff, float eps, int dtype, void* workspace,
                           size_t workspace_bytes, void* stream);
size_t beacon_llama_block_workspace_size(int64_t batch, int64_t seq, int64_t d_model, int64_t heads,
                                         int64_t kv_heads, int64_t head_dim, int64_t d_ff, int dtype);

/* The same block with both RMSNorms folded into the GEMMs that consume them (six
 * launches and a 4-byte-per-row memset, no normalised activations written or read):
 * w_qkv_folded = diag(attn_norm) . w_qkv, w_gate_folded = diag(ffn_norm) . w_gate,
 * w_up_folded = diag(ffn_norm) . w_up, each made once per weight version with
 * beacon_rmsnorm_fold_weight.  The first norm's statistic is one read of x; the second's
 * is summed in the output projection's epilogue from the h it stores.  Same workspace. */
int beacon_llama_block_fwd_folded(void* out, const void* x, const void* w_qkv_folded, const void* w_o,
                                  const void* w_gate_folded, const void* w_up_folded, const void* w_down,
                                  int64_t batch, int64_t seq, int64_t d_model, int64_t heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t d_ff, float eps, int dtype, void* workspace,
                                  size_t workspace_bytes, void* stream);

/* ---- position rotation and paged cache (no reference counterpart) ----------
 * The reference has no position encoding and no key/value cache; these entries stand between
 * linear_fwd (the fused QKV projection) and attention in training, and make the block run on new
 * tokens after earlier ones in serving.
 *
 * Rotation table, float32 [positions, rot_dim]: row t holds cos(t theta^(-2i / rot_dim)) for
 * i < rot_dim / 2, then the sines; evaluated in 64 bits.  Made once; any table of that layout
 * (scaled or extended rotations) serves the entries below. */
int beacon_rope_table(float* table, int64_t positions, int64_t rot_dim, double theta, void* stream);

/* Per-head RMS norm of queries and keys, the position rotation and the layout change in one pass.
 * qkv: batch * seq token rows, qkv_stride elements apart, of q_heads + 2 kv_heads heads of head_dim
 * (queries, keys, values); q [batch, q_heads, seq, head_dim]; k, v [batch, kv_heads, seq, head_dim]
 * (v NULL: the value heads are not copied).  For a query or key head x with gain g [head_dim]:
 *   z = g x / sqrt(mean x^2 + eps)   (gain NULL: z = x, no norm),
 *   y_a = z_a c_i - z_b s_i,  y_b = z_b c_i + z_a s_i,  y_d = z_d for d >= rot_dim,
 * (a, b) = (i, i + rot_dim / 2), or (2i, 2i + 1) when `interleaved`; (c, s) from the table's row of the
 * token's position: positions [batch * seq], or the place in the sequence when NULL.  rot_dim 0: no
 * rotation (table may be NULL).  A position outside the table is not followed: the token's query and
 * key rows are zeros (their gradients too) and the device fault word records code 3.
 * head_dim up to 256, f32 or bf16 (one rounding, at the store).  16-byte aligned pointers and rows, a
 * head_dim of 64, 128 or 256 and rot_dim % 16 == 0 take the vectorised kernels. */
int beacon_qk_norm_rope_fwd(void* q, void* k, void* v, const void* qkv, int64_t qkv_stride, const void* q_gain,
                            const void* k_gain, const float* table, int64_t table_positions,
                            const int32_t* positions, int64_t batch, int64_t seq, int64_t q_heads,
                            int64_t kv_heads, int64_t head_dim, int64_t rot_dim, int interleaved, float eps,
                            int dtype, void* stream);

/* Its backward, the statistics formed again from qkv (whose value columns are not read):
 *   dz = the rotation of dy by the opposite angle, dgain = sum over tokens and heads of dz x / r,
 *   e = g dz, dx = e / r - x sum(e x) / (head_dim r^3)   (dx = dz without a gain).
 * dqkv rows lie dqkv_stride elements apart; dv NULL leaves their value columns as they are.
 * dq_gain, dk_gain [head_dim] may be NULL; their sums are kept in float32 and added in a fixed order
 * (results do not depend on timing).  Workspace of beacon_qk_norm_rope_bwd_workspace_size bytes, needed only
 * for gain gradients, or NULL for the library's; a captured call needs its own (below). */
int beacon_qk_norm_rope_bwd(void* dqkv, int64_t dqkv_stride, void* dq_gain, void* dk_gain, const void* dq,
                            const void* dk, const void* dv, const void* qkv, int64_t qkv_stride,
                            const void* q_gain, const void* k_gain, const float* table, int64_t table_positions,
                            const int32_t* positions, int64_t batch, int64_t seq, int64_t q_heads,
                            int64_t kv_heads, int64_t head_dim, int64_t rot_dim, int interleaved, float eps,
                            int dtype, void* workspace, size_t workspace_bytes, void* stream);
size_t beacon_qk_norm_rope_bwd_workspace_size(int64_t head_dim);

/* Paged caches.  k_cache, v_cache: num_pages pages of page_size tokens, any layout with dense rows:
 * element (page, KV head, token, d) at page * page_stride + head * head_stride + token * token_stride
 * + d (the same strides for both).  Sequence s of `seqs` owns the token rows [cu_q[s], cu_q[s + 1]) of the
 * token-major tensors and kv_lens[s] cached tokens, the new ones included and last; its token j
 * sits in page page_table[s * table_stride + j / page_size] (max_pages entries per row; entries past the
 * last used page are not read).  cu_q, kv_lens and page_table are int32 in device memory and are read on
 * the stream: no host copy, so the calls can be captured.  A captured call needs a workspace of its own, which
 * lives as long as its graph: the library's buffer is freed when a later call needs a larger one, so NULL
 * is refused with InvalidLaunchConfig on a stream that is being captured.  A page index outside the cache is not
 * followed (its tokens are not written, its keys and values read as zeros), and lengths that reach
 * past the tensors are cut; with a cu_q that decreases attention does nothing and the tokens that it
 * gives no place are not written.  All record fault code 3.  Token rows that no sequence owns are ignored.
 *
 * qk_norm_rope_append: beacon_qk_norm_rope_fwd for new tokens, the queries written token-major
 * [tokens, q_heads, head_dim], keys and values into the pages.  Tokens rotate by their place j in the
 * sequence, or by positions [tokens]. */
int beacon_qk_norm_rope_append(void* q, void* k_cache, void* v_cache, const void* qkv, int64_t qkv_stride,
                               const void* q_gain, const void* k_gain, const float* table,
                               int64_t table_positions, const int32_t* positions, const int32_t* cu_q,
                               const int32_t* kv_lens, const int32_t* page_table, int64_t tokens, int64_t seqs,
                               int64_t max_pages, int64_t table_stride, int64_t num_pages, int64_t page_size,
                               int64_t page_stride, int64_t head_stride, int64_t token_stride, int64_t q_heads,
                               int64_t kv_heads, int64_t head_dim, int64_t rot_dim, int interleaved, float eps,
                               int dtype, void* stream);

/* Attention of the new tokens over the cache: q [tokens, q_heads, head_dim] (rows q_stride elements
 * apart, dense heads), out [tokens, q_heads, head_dim], lse [tokens, q_heads] float32 (may be NULL).  New
 * token i of a sequence sits at p = kv_len - q_len + i and sees the keys j <= p (causal) or every one:
 * out = softmax(q k^T / sqrt(head_dim)) v, lse = natural-log logsumexp; a token that sees no key gets out
 * 0 and lse -inf.  A token that sees a score of NaN or +inf, or scores of -inf only, gets out NaN and lse NaN,
 * +inf or -inf (the logarithm of its sum).  Query head h reads KV head h / (q_heads / kv_heads).  Values in
 * cache slots at or beyond kv_lens never reach a result, NaN included; the values of cached keys that a token does not see are
 * multiplied by 0, so NaN or infinity among them can reach it.  max_q: the largest number of new tokens of a
 * sequence if known, else 0 (the mean stands for it: a batch of single tokens with one prompt of 64 took 179 us
 * so, 149 with it); it only chooses between kernels.  head_dim 16, 32, 64 or 128; bf16 or f32
 * (exact fp32 products).  Workspace of beacon_paged_attention_workspace_size bytes, 32-byte aligned
 * (partial rows of work split along the keys; it may hold anything), or NULL for the library's. */
int beacon_paged_attention_fwd(void* out, float* lse, const void* q, int64_t q_stride, const void* k_cache,
                               const void* v_cache, const int32_t* cu_q, const int32_t* kv_lens,
                               const int32_t* page_table, int64_t tokens, int64_t seqs, int64_t max_q,
                               int64_t max_pages, int64_t table_stride, int64_t num_pages, int64_t page_size,
                               int64_t page_stride, int64_t head_stride, int64_t token_stride, int64_t q_heads,
                               int64_t kv_heads, int64_t head_dim, int causal, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream);
size_t beacon_paged_attention_workspace_size(int64_t head_dim, int dtype);

/* beacon_llama_block_fwd on new tokens of sequences with cached keys and values: x, out [tokens, d_model],
 * the tokens of all sequences one after another as cu_q says, prompt chunks and single tokens mixed as they
 * come.  Per-head norms (q_gain, k_gain [head_dim], NULL: none) and the rotation (rope_table NULL with
 * rot_dim 0: none) act on queries and keys before the new keys and values enter the pages; attention is
 * causal over the whole cache.  bf16; the other conditions are beacon_llama_block_fwd's and
 * beacon_paged_attention_fwd's.  Scratch: beacon_llama_block_paged_workspace_size bytes, 32-byte aligned, or NULL
 * for the library's.  Nothing is read back, so a step can be captured, with a workspace of its own.  Rows of out for tokens that no sequence owns are
 * undefined. */
int beacon_llama_block_paged_fwd(void* out, const void* x, const void* attn_norm, const void* w_qkv,
                                 const void* q_gain, const void* k_gain, const void* w_o, const void* ffn_norm,
                                 const void* w_gate, const void* w_up, const void* w_down, const float* rope_table,
                                 int64_t table_positions, int64_t rot_dim, int interleaved, void* k_cache,
                                 void* v_cache, const int32_t* cu_q, const int32_t* kv_lens,
                                 const int32_t* page_table, int64_t tokens, int64_t seqs, int64_t max_q,
                                 int64_t max_pages, int64_t table_stride, int64_t num_pages, int64_t page_size,
                                 int64_t page_stride, int64_t head_stride, int64_t token_stride, int64_t d_model,
                                 int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t d_ff, float eps,
                                 int dtype, void* workspace, size_t workspace_bytes, void* stream);
size_t beacon_llama_block_paged_workspace_size(int64_t tokens, int64_t d_model, int64_t heads, int64_t kv_heads,
                                               int64_t head_dim, int64_t d_ff, int dtype);

/* ---- elementwise: crates/beacon-cuda/src/elementwise.rs -------------------- */

/* residual_add (elementwise.rs:47-55): out = a + b */
int beacon_residual_add_fwd(void* out, const void* a, const void* b, int64_t n, int dtype, void* stream);
/* residual_add_backward (elementwise.rs:57-65): d_a = d_b = d_out */
int beacon_residual_add_bwd(void* d_a, void* d_b, const void* d_out, int64_t n, int dtype, void* stream);
/* cast (elementwise.rs:120-128) with the reference's rounding rules (dtype.rs:58-66, 163-195). */
int beacon_cast(void* dst, const void* src, int64_t n, int kind, void* stream);

/* embedding_lookup (elementwise.rs:67-80): out[t, :] = table[indices[t], :], u32 indices.
 * embedding_backward (elementwise.rs:82-95): d_table[indices[t], :] += d_out[t, :] (atomic
 * adds; d_table is accumulated into, as its ReadWrite access in the reference's test says).
 * `vocab` (table rows) bounds the indices: an index >= vocab is not followed -- the forward
 * writes a zero row, the backward skips the token -- and the device fault word records code 3
 * (read it with beacon_device_status).  f32 or bf16 (bf16 adds round at every add). */
int beacon_embedding_lookup_fwd(void* out, const void* table, const uint32_t* indices, int64_t tokens, int64_t dim,
                                int64_t vocab, int dtype, void* stream);
int beacon_embedding_lookup_bwd(void* d_table, const void* d_out, const uint32_t* indices, int64_t tokens,
                                int64_t dim, int64_t vocab, int dtype, void* stream);

/* dropout_forward (elementwise.rs:97-108): element i is kept when u_i >= p, with
 * u_i = (splitmix64(seed, i) >> 40) / 2^24 (SplitMix64: z = seed + (i + 1) * 0x9E3779B97F4A7C15,
 * then the usual two xor-shift-multiply rounds), so the mask depends on (seed, i) only.
 * mask[i] = 1 / (1 - p) rounded to dtype for a kept element, 0 for a dropped one;
 * out = input * mask.  dropout_backward (elementwise.rs:110-118, no p): d_in = d_out * mask.
 * p >= 1 drops everything.  f32 or bf16; mask has the data type. */
int beacon_dropout_fwd(void* out, const void* input, void* mask, int64_t n, float p, uint64_t seed, int dtype,
                       void* stream);
int beacon_dropout_bwd(void* d_in, const void* d_out, const void* mask, int64_t n, int dtype, void* stream);

/* ---- arena launcher: the KernelLauncher::launch boundary ------------------
 * crates/beacon-cuda/src/runtime.rs:31-47 (Launcher::launch) and
 * crates/beacon-cuda/src/launcher.rs:21-63 (KernelArg = byte offset into one arena).
 * A Rust `Launcher` implements KernelLauncher::launch by forwarding here; the
 * typed traits' shapes, which they drop before launch, travel in `scalars`, in
 * this order per kernel ID (args in the typed trait's order):
 *   matmul_fwd/_bwd, linear_fwd/_bwd          m, k, n, dtype
 *   attention_adjoint_fwd/_bwd                batch, heads, seqlen, head_dim, causal, dtype[, kv_heads]
 *   rmsnorm_ / layernorm_adjoint_fwd/_bwd     tokens, dim, dtype[, eps as float32 bits]
 *   swiglu_adjoint_fwd/_bwd                   tokens, d_model, d_ff, dtype
 *   residual_add_fwd/_bwd                     n, dtype
 *   cast_*                                    n
 *   embedding_lookup_fwd/_bwd                 tokens, dim[, dtype]  (vocab = table extent / row)
 *   dropout_fwd                               n, p as float32 bits, seed[, dtype]
 *   dropout_bwd                               n[, dtype]                                   */
typedef struct beacon_arena beacon_arena;

typedef struct beacon_kernel_arg {
    uint64_t offset;     /* byte offset into the arena */
    uint64_t len_bytes;  /* extent, checked against the arena and the shapes */
    int32_t access;      /* 0 Read, 1 Write, 2 ReadWrite (launcher.rs:14-19) */
} beacon_kernel_arg;

/* Creates an arena of `bytes` device memory on `device` (256-byte aligned
 * regions are the caller's business, crates/beacon-core/src/arena.rs:7). */
beacon_arena* beacon_arena_create(int device, uint64_t bytes);
void beacon_arena_destroy(beacon_arena* arena);

/* The launcher's workspace (crates/beacon-cuda/src/runtime.rs:6-48 keeps one Launcher per
 * device; "kernels never allocate"): `bytes` of device memory owned by the arena, made once
 * at set-up (a second call replaces it, after a device synchronisation).  beacon_launch
 * hands it to every kernel ID that needs scratch (the attention, RMSNorm, LayerNorm and
 * SwiGLU backward, linear_bwd's dbias, the SwiGLU forward) and never allocates: when the
 * workspace is missing or too small the launch fails with BEACON_ERR_OUT_OF_MEMORY
 * ("requested / available").  Size it with the beacon_*_workspace_size functions. */
int beacon_workspace_create(beacon_arena* arena, uint64_t bytes);
void* beacon_arena_base(beacon_arena* arena);
uint64_t beacon_arena_size(beacon_arena* arena);

/* Dispatch by kernel ID string (the adjoint-table launcher names plus the
 * elementwise IDs).  `scalars` carries the dropped shapes, then dtype. */
int beacon_launch(beacon_arena* arena, const char* kernel, const beacon_kernel_arg* args, size_t nargs,
                  const int64_t* scalars, size_t nscalars, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* BEACON_CUDA_H */
