/*
 * kda.h -- C ABI of the kda-b200 fused-operator library (libkda.so, sm_100a).
 *
 * One entry point per operator of the reference's NKIBench operator set
 * (Jerry2423/kda-for-trainium).  Each replaces the reference's per-operator
 * numpy `forward(...)` / NKI `kernel(...)` pair: arguments keep the forward's
 * parameter names and order, in natural (untiled) row-major layout, followed
 * by sizes, an optional caller-owned workspace, and the CUDA stream.
 * Around them: fp32-accuracy variants of the contractions (`*_f32`), the
 * training-side neighbours of the path (backward kernels, a multi-tensor
 * AdamW, a fused ZeRO-1 step over NVLink with its CUDA IPC helpers).
 *
 * Conventions
 *   - All pointers are device pointers owned by the caller.  bf16 tensors are
 *     passed as `const void*` (raw bf16 storage); fp32 tensors as float*.
 *   - Calls are asynchronous and stream-ordered on `stream` (a cudaStream_t,
 *     passed as void*; NULL = legacy default stream).  No call synchronises
 *     the device or allocates memory (kda_ipc_open maps a peer's existing
 *     allocation).  Calls are reentrant: concurrent calls
 *     on different streams or devices are safe when they do not share output
 *     or workspace buffers.
 *   - Every entry point returns a kda_status; no C++ exception crosses the
 *     ABI.  kda_last_error() gives the calling thread's detail message.
 *   - Kernels bound every internal wait; a wait that expires writes a code to
 *     a device error word that kda_device_error() reads after the stream is
 *     synchronised.  The local-attention kernels report a position or length
 *     outside its table or cache there too, with the value 8.
 *   - Ops that need scratch memory take (workspace, workspace_bytes); the
 *     required size comes from the matching *_workspace_size() query.
 */
#ifndef KDA_H_
#define KDA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KDA_ABI_VERSION 1

typedef enum kda_status {
  KDA_OK = 0,
  KDA_INVALID_ARG = 1,  /* null pointer, bad dimension, too-small workspace */
  KDA_UNSUPPORTED = 2,  /* shape / alignment outside the kernel's contract   */
  KDA_CUDA_ERROR = 3,   /* launch or driver failure (cudaGetLastError)       */
  KDA_TIMEOUT = 4       /* a bounded device wait expired (kda_device_error)  */
} kda_status;

/* ------------------------------------------------------------- library -- */
int kda_abi_version(void);
const char* kda_status_string(kda_status s);
/* Detail message of the last non-OK status returned on this thread. */
const char* kda_last_error(void);
/* Reads (and with clear != 0 resets) the OR of the device error words of the
 * current device.  *word == 0 (KDA_OK): no kernel reported anything.  A word
 * of 8 (KDA_INVALID_ARG): a position or length lay outside its table or cache.
 * Any other (KDA_TIMEOUT): a kernel's wait expired.
 * Synchronous with respect to the device (cudaMemcpyFromSymbol). */
kda_status kda_device_error(unsigned* word, int clear);

/* ------------------------------------------------------ elementwise ops -- */

/* silu: y = x / (1 + exp(-x)), fp32, n elements.
 * Replaces silu forward(x) (prompts/_gen_prompts.py:19-33) and the NKI kernel
 * workspaces/silu/runs/silu_v3_s7.py:31-71. */
kda_status kda_silu_f32(const float* x, float* y, int64_t n, void* stream);

/* rope_single_freq_apply: half-split rotation over the leading axis.
 * x_in (d_head, s) row-major, cos/sin (d_head/2, s), out (d_head, s):
 *   out[:h] = x0*cos - x1*sin ; out[h:] = x0*sin + x1*cos   (h = d_head/2)
 * Replaces rope_single_freq_apply forward(x_in, cos, sin)
 * (workspaces/rope_single_freq_apply/runs/rope_v1.py:5-8, kernel :33). */
kda_status kda_rope_single_freq_apply_f32(const float* x_in, const float* cos, const float* sin, float* out,
                                          int64_t d_head, int64_t s, void* stream);

/* adamw: one AdamW step with the reference constants (lr 0.01, beta1 0.9,
 * beta2 0.999, weight decay 1e-5, eps 1e-8, bias-correction 1000 on v):
 *   m' = .9m + .1g ; v' = .999v + .001g^2 ;
 *   theta_out = theta - 1e-5 theta - .01 m'/(sqrt(1000 v') + 1e-8)
 * If update_state != 0, m and v are overwritten with m', v' (in place).
 * Replaces adamw forward(theta, g, m, v) (prompts/_gen_prompts.py:227-228,
 * workspaces/adamw/runs/adamw_v1.py:5-11; kernel adamw_v2_ch1824.py:51). */
kda_status kda_adamw_f32(const float* theta, const float* g, float* m, float* v, float* theta_out, int64_t n,
                         int update_state, void* stream);

/* adamw_multi: the AdamW step over a list of `count` fp32 tensors, in place
 * (theta, m, v updated; g read), one launch per 48 tensors.  Decoupled weight
 * decay and bias correction at `step` (>= 1):
 *   m' = b1 m + (1-b1) g ; v' = b2 v + (1-b2) g^2 ;
 *   theta' = (theta - lr wd theta) - lr/(1-b1^step) m' / (sqrt(v'/(1-b2^step)) + eps)
 * Hyperparameters in double.  lr 1e-3, betas (0.9, 0.999), eps 1e-8, wd 1e-2,
 * step 1 is exactly the adamw forward above (workspaces/adamw/runs/adamw_v1.py:5-11),
 * applied to many tensors at once: the multi-tensor form of the step that
 * follows it in training. */
kda_status kda_adamw_multi_f32(float* const* theta, const float* const* g, float* const* m, float* const* v,
                               const int64_t* n, int count, double lr, double beta1, double beta2, double eps,
                               double weight_decay, int64_t step, void* stream);

/* CUDA IPC for the ZeRO-1 step: export a device pointer as (handle, offset
 * into its allocation), open a peer's export in this process (mapped with
 * peer access; no multicast), close it again.  The handle is
 * kda_ipc_handle_size() bytes.  No reference counterpart: the reference has
 * no multi-device code (the plumbing of adamw's training-step neighbour). */
size_t kda_ipc_handle_size(void);
kda_status kda_ipc_export(const void* ptr, void* handle, int64_t* offset);
kda_status kda_ipc_open(const void* handle, int64_t offset, void** ptr);
kda_status kda_ipc_close(void* ptr, int64_t offset);

/* zero1_adamw: one fused ZeRO-1 step for this rank's shard [shard_off,
 * shard_off + shard_len) of flat fp32 buffers replicated on `world` ranks
 * (<= 8): g = (1/world) sum_r grads[r][shard] (peer loads), AdamW as
 * kda_adamw_multi_f32 on params[rank][shard] with this rank's moments m, v
 * (shard_len elements), and the new values stored into params[r][shard] of
 * every rank (peer stores).  grads / params hold every rank's buffer address
 * in this process (its own, and kda_ipc_open'ed peers).  shard_off and
 * shard_len multiples of 4, all buffers 16-byte aligned.  The caller orders
 * the step: every rank's gradients complete before any rank launches, and no
 * rank touches its buffers again until every rank's launch has completed
 * (e.g. a one-element all-reduce on the stream before and after).  The
 * reduce-scatter -> adamw -> all-gather around the adamw forward
 * (workspaces/adamw/runs/adamw_v1.py:5-11) as one kernel. */
kda_status kda_zero1_adamw_f32(const float* const* grads, float* const* params, int world, int rank,
                               int64_t shard_off, int64_t shard_len, float* m, float* v, double lr, double beta1,
                               double beta2, double eps, double weight_decay, int64_t step, void* stream);

/* ------------------------------------------------------ selective scan -- */

/* mamba: h_t = exp(dt_t * A) h_{t-1} + dt_t B_t x_t ; y_t = C_t . h_t + D x_t
 * fp32 state (h_0 = 0), d_state == 16.
 * Batched channels-last layout: delta (dt) and u (x) are (batch, seqlen,
 * d_inner) with element (b,t,d) at b*ld_b + t*ld_t + d*ld_d (element
 * strides); a (A) is (d_inner, 16) contiguous; b (B) and c (C) are
 * (batch, seqlen, 16) with element (b,t,n) at b*bc_ld_b + t*bc_ld_t + n*bc_ld_n;
 * D is (d_inner,) or NULL; y has the strides of delta.
 * u_bf16 != 0: u is bf16 storage, else fp32.  y_bf16 != 0: y is bf16, else fp32.
 * The reference's 2-D form -- delta, u (C, M); a (C, S); b, c (S, M) -- is
 * batch 1, ld_t = 1, ld_d = M, bc_ld_t = 1, bc_ld_n = M.
 * When batch * d_inner is too small to fill the GPU, time is split into
 * chunks scanned in parallel; their summaries need the workspace that
 * kda_mamba_scan_workspace_size() reports (0 bytes when no chunking is used).
 * Replaces mamba forward(delta, u, a, b, c) (workspaces/mamba/docs/
 * draft-phase1.md:22-29; kernel workspaces/mamba/runs/mamba_v4_s4unroll.py:8). */
size_t kda_mamba_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t d_inner, int64_t d_state);
kda_status kda_mamba_scan(const void* delta, const void* u, const float* a, const float* b, const float* c,
                          const float* D, void* y, int64_t batch, int64_t seqlen, int64_t d_inner,
                          int64_t d_state, int64_t ld_b, int64_t ld_t, int64_t ld_d, int64_t bc_ld_b,
                          int64_t bc_ld_t, int64_t bc_ld_n, int u_bf16, int y_bf16, void* workspace,
                          size_t workspace_bytes, void* stream);

/* mamba_scan_noalloc: the same scan as kda_mamba_scan, for callers that
 * cannot allocate device memory -- a host binding that is handed only the
 * input and output buffers by its framework, or code that must not call
 * cudaMalloc because it can synchronise the device.  It has no counterpart in
 * the reference.  When the time axis is split into chunks, the chunk summaries
 * go to a fixed 1 MiB array that every GPU loading the library holds until
 * the process exits; shapes needing more (kda_mamba_scan_workspace_size() >
 * 1 MiB) are rejected with KDA_UNSUPPORTED.  The first call on each device
 * looks up that array's device address (cudaGetSymbolAddress), so make it
 * before any stream capture.  All calls share the array: calls that overlap
 * on the GPU (other streams, other threads) race and must be serialised by
 * the caller.  No memory is allocated or freed.  Arguments as kda_mamba_scan
 * without the workspace. */
kda_status kda_mamba_scan_noalloc(const void* delta, const void* u, const float* a, const float* b,
                                  const float* c, const float* D, void* y, int64_t batch, int64_t seqlen,
                                  int64_t d_inner, int64_t d_state, int64_t ld_b, int64_t ld_t, int64_t ld_d,
                                  int64_t bc_ld_b, int64_t bc_ld_t, int64_t bc_ld_n, int u_bf16, int y_bf16,
                                  void* stream);

/* ---------------------------------------------------------- contractions --
 * bf16 operands, fp32 accumulation in tensor memory (tcgen05), bf16 output
 * unless stated.  Row strides must be multiples of 16 bytes (TMA), and the
 * base pointers 16-byte aligned. */

/* matmul: out (M,N) = lhs (M,K) @ rhs (K,N).
 * Replaces matmul forward(lhs, rhs) (workspaces/matmul/runs/offline_bf16_split_sim.py:137-139;
 * kernel workspaces/matmul/runs/matmul_v3_bf16_split.py:11). */
kda_status kda_matmul_bf16(const void* lhs, const void* rhs, void* out, int64_t M, int64_t K, int64_t N,
                           void* stream);

/* matmul, fp32 in / fp32 out at fp32 accuracy on the bf16 tensor core: each
 * operand is split into bf16 hi + lo (in the workspace) and
 * out = hi.hi + hi.lo + lo.hi is accumulated in fp32 -- the reference's
 * bf16 split of fp32 operands (workspaces/matmul/runs/matmul_v3_bf16_split.py:14-24;
 * forward workspaces/matmul/runs/offline_bf16_split_sim.py:137-139). */
size_t kda_matmul_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_matmul_f32(const float* lhs, const float* rhs, float* out, int64_t M, int64_t K, int64_t N,
                          void* workspace, size_t workspace_bytes, void* stream);

/* transpose_matmul: out (M,N) = lhs^T @ rhs, lhs stored (K,M).
 * Replaces transpose_matmul forward(lhs, rhs)
 * (workspaces/transpose_matmul/runs/offline_bf16_split_sim.py:101-104; kernel
 * workspaces/transpose_matmul/runs/tmm_v3_mblk16_bf16_split.py:11). */
kda_status kda_transpose_matmul_bf16(const void* lhs, const void* rhs, void* out, int64_t M, int64_t K,
                                     int64_t N, void* stream);

/* transpose_matmul, fp32 in / fp32 out at fp32 accuracy: the bf16 hi + lo
 * split of kda_matmul_f32 with lhs (K,M) read MN-major
 * (workspaces/transpose_matmul/runs/tmm_v3_mblk16_bf16_split.py:11, the
 * reference's bf16-split kernel; forward
 * workspaces/transpose_matmul/runs/offline_bf16_split_sim.py:101-104). */
size_t kda_transpose_matmul_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_transpose_matmul_f32(const float* lhs, const float* rhs, float* out, int64_t M, int64_t K,
                                    int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* bmm: out[b] (M,N) = lhs[b] (M,K) @ rhs[b] (K,N), b < batch.
 * Replaces bmm forward(lhs, rhs) (workspaces/bmm/runs/offline_bf16_split_sim.py:102-117;
 * kernel workspaces/bmm/runs/bmm_v2.py:11). */
kda_status kda_bmm_bf16(const void* lhs, const void* rhs, void* out, int64_t batch, int64_t M, int64_t K,
                        int64_t N, void* stream);

/* bmm, fp32 in / fp32 out at fp32 accuracy: both operands split into bf16
 * hi + lo once for the whole batch, then one three-pass GEMM per entry
 * (forward workspaces/bmm/runs/offline_bf16_split_sim.py:102-104, whose
 * bf16-split product it reproduces). */
size_t kda_bmm_f32_workspace_size(int64_t batch, int64_t M, int64_t K, int64_t N);
kda_status kda_bmm_f32(const float* lhs, const float* rhs, float* out, int64_t batch, int64_t M, int64_t K,
                       int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* bmm_softmax: out[b] = softmax over the last axis of lhs[b] @ rhs[b]
 * (max-shifted, fp32 scores and statistics, bf16 out).
 * Replaces bmm_softmax forward(lhs, rhs) (prompts/_gen_prompts.py:170-177;
 * kernel workspaces/bmm_softmax/runs/bmm_softmax_v4.py:11-27). */
kda_status kda_bmm_softmax_bf16(const void* lhs, const void* rhs, void* out, int64_t batch, int64_t M,
                                int64_t K, int64_t N, void* stream);

/* bmm_softmax, fp32 in / fp32 out at fp32 accuracy: kda_bmm_f32, then a
 * max-shifted fp32 row softmax in place (the spec's fp32 forward,
 * prompts/_gen_prompts.py:170-177). */
size_t kda_bmm_softmax_f32_workspace_size(int64_t batch, int64_t M, int64_t K, int64_t N);
kda_status kda_bmm_softmax_f32(const float* lhs, const float* rhs, float* out, int64_t batch, int64_t M, int64_t K,
                               int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* rmsnorm_matmul: out = (x / sqrt(mean_k x^2 + eps) * g) @ w ; g may be NULL
 * (the reference: no gamma, eps = 0).  x (M,K), w (K,N), g (K,) fp32.
 * Replaces rmsnorm_matmul forward(x, w)
 * (workspaces/rmsnorm_matmul/runs/offline_bf16_split_sim.py:83-93; kernel
 * workspaces/rmsnorm_matmul/runs/rmsnorm_matmul_v4_bf16_split.py:11). */
size_t kda_rmsnorm_matmul_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_rmsnorm_matmul_bf16(const void* x, const void* w, const float* g, float eps, void* out, int64_t M,
                                   int64_t K, int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* rmsnorm_matmul, fp32 x / w / out at fp32 accuracy: a row kernel normalises
 * x in fp32 and writes the bf16 hi + lo split of the normalised rows, then the
 * three-pass split GEMM (the reference forward in fp32,
 * workspaces/rmsnorm_matmul/runs/offline_bf16_split_sim.py:83-93, and its
 * bf16-split kernel workspaces/rmsnorm_matmul/runs/rmsnorm_matmul_v4_bf16_split.py:11). */
size_t kda_rmsnorm_matmul_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_rmsnorm_matmul_f32(const float* x, const float* w, const float* g, float eps, float* out, int64_t M,
                                  int64_t K, int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* rmsnorm_matmul backward: the gradients of out = a @ w, a = x r g,
 * r = 1 / sqrt(mean_k x^2 + eps), given dy (M,N):
 *   dx (M,K) bf16 = r (dA g - xn mean_k(dA g xn)),  xn = x r,  dA = dy @ w^T (fp32)
 *   dw (K,N) bf16 = a^T @ dy  (a recomputed as the forward's bf16 operand)
 *   dg (K,)  fp32 = sum_m dA xn  (written iff g is given; deterministic order)
 * dy, x, w bf16; g fp32 or NULL.  The training-side caller of rmsnorm_matmul
 * forward (workspaces/rmsnorm_matmul/runs/offline_bf16_split_sim.py:83-93); the
 * reference has no backward (its operators are forward-only). */
size_t kda_rmsnorm_matmul_backward_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_rmsnorm_matmul_backward_bf16(const void* dy, const void* x, const void* w, const float* g, float eps,
                                            void* dx, void* dw, float* dg, int64_t M, int64_t K, int64_t N,
                                            void* workspace, size_t workspace_bytes, void* stream);

/* add_rmsnorm_matmul: a = x + z ; out = (a / sqrt(mean_k a^2 + eps) * g) @ w.
 * x, z (M,K) bf16, w (K,N) bf16, g (K,) fp32.
 * Replaces add_rmsnorm_matmul forward(x, w, eps, z, g)
 * (workspaces/add_rmsnorm_matmul/runs/offline_bf16_split_sim.py:97-106; kernel
 * workspaces/add_rmsnorm_matmul/runs/add_rmsnorm_matmul_v3_bf16_split.py:9). */
size_t kda_add_rmsnorm_matmul_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_add_rmsnorm_matmul_bf16(const void* x, const void* w, float eps, const void* z, const float* g,
                                       void* out, int64_t M, int64_t K, int64_t N, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* add_rmsnorm_matmul, fp32 x / z / w / out at fp32 accuracy (as
 * kda_rmsnorm_matmul_f32 on a = x + z;
 * workspaces/add_rmsnorm_matmul/runs/offline_bf16_split_sim.py:97-106). */
size_t kda_add_rmsnorm_matmul_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_add_rmsnorm_matmul_f32(const float* x, const float* w, float eps, const float* z, const float* g,
                                      float* out, int64_t M, int64_t K, int64_t N, void* workspace,
                                      size_t workspace_bytes, void* stream);

/* matmul_add_rmsnorm: y = x @ w + z ; out = y * g / sqrt(mean_n y^2 + eps).
 * x (M,K), w (K,N), z (M,N) bf16; g (N,) fp32; out (M,N) bf16.
 * Replaces matmul_add_rmsnorm forward(x, w, eps, z, g)
 * (workspaces/matmul_add_rmsnorm/runs/offline_bf16_split_sim.py:111-115; kernel
 * workspaces/matmul_add_rmsnorm/runs/matmul_add_rmsnorm_v2_bf16_split.py:9). */
size_t kda_matmul_add_rmsnorm_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_matmul_add_rmsnorm_bf16(const void* x, const void* w, float eps, const void* z, const float* g,
                                       void* out, int64_t M, int64_t K, int64_t N, void* workspace,
                                       size_t workspace_bytes, void* stream);

/* matmul_add_rmsnorm, fp32 in / out at fp32 accuracy: the three-pass split
 * GEMM writes x @ w into out, a row kernel adds z and normalises in place
 * (workspaces/matmul_add_rmsnorm/runs/offline_bf16_split_sim.py:111-115). */
size_t kda_matmul_add_rmsnorm_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_matmul_add_rmsnorm_f32(const float* x, const float* w, float eps, const float* z, const float* g,
                                      float* out, int64_t M, int64_t K, int64_t N, void* workspace,
                                      size_t workspace_bytes, void* stream);

/* swiglu: out (M,K) = (silu(x @ w_gate) * (x @ w_up)) @ w_down.
 * x (M,K), w_up / w_gate (K,N), w_down (N,K), all bf16; the intermediate h
 * (M,N) is stored once in the workspace as bf16.
 * Replaces swiglu forward(x, w_up, w_down, w_gate)
 * (workspaces/swiglu/runs/offline_bf16_split_sim.py:87-97; kernel
 * workspaces/swiglu/runs/swiglu_v3_mblock.py:47). */
size_t kda_swiglu_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_swiglu_bf16(const void* x, const void* w_up, const void* w_down, const void* w_gate, void* out,
                           int64_t M, int64_t K, int64_t N, void* workspace, size_t workspace_bytes,
                           void* stream);

/* swiglu, fp32 in / out at fp32 accuracy: [gate | up] in one three-pass GEMM
 * (fp32, in the workspace), h = silu(gate) * up in fp32 written as its bf16
 * hi + lo split, then h @ w_down (the reference forward with its fp32 h,
 * workspaces/swiglu/runs/offline_bf16_split_sim.py:87-97). */
size_t kda_swiglu_f32_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_swiglu_f32(const float* x, const float* w_up, const float* w_down, const float* w_gate, float* out,
                          int64_t M, int64_t K, int64_t N, void* workspace, size_t workspace_bytes, void* stream);

/* swiglu backward: the gradients of out = (silu(x w_gate) * (x w_up)) w_down
 * given dout (M,K): dx (M,K), dw_up / dw_gate (K,N), dw_down (N,K), all bf16
 * (fp32 accumulation; g = x w_gate and u = x w_up recomputed; N is d_ff):
 *   dh = dout w_down^T ; dg = dh u silu'(g) ; du = dh silu(g)
 *   dw_down = h^T dout ; dw_gate = x^T dg ; dw_up = x^T du ; dx = dg w_gate^T + du w_up^T
 * The training-side caller of swiglu forward
 * (workspaces/swiglu/runs/offline_bf16_split_sim.py:87-97); the reference has no
 * backward. */
size_t kda_swiglu_backward_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_swiglu_backward_bf16(const void* dout, const void* x, const void* w_up, const void* w_down,
                                    const void* w_gate, void* dx, void* dw_up, void* dw_down, void* dw_gate,
                                    int64_t M, int64_t K, int64_t N, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* swiglu forward of a training step: out as kda_swiglu_bf16 computes it, but
 * unfused -- g = x w_gate and u = x w_up (bf16, M x N) are written to the
 * caller's buffers, h = silu(g) * u (from the bf16 g, u) goes through the
 * workspace (kda_swiglu_gu_workspace_size()) into out = h w_down -- so that
 * kda_swiglu_backward_saved_bf16 need not recompute g and u.  Same reference
 * forward as kda_swiglu_bf16 (workspaces/swiglu/runs/offline_bf16_split_sim.py:87-97);
 * the reference keeps no activations, so no counterpart for g and u. */
size_t kda_swiglu_gu_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_swiglu_gu_bf16(const void* x, const void* w_up, const void* w_down, const void* w_gate, void* out,
                              void* g, void* u, int64_t M, int64_t K, int64_t N, void* workspace,
                              size_t workspace_bytes, void* stream);

/* swiglu backward from the saved g and u of kda_swiglu_gu_bf16: the same
 * gradients as kda_swiglu_backward_bf16 without its two recomputing GEMMs
 * (smaller workspace, kda_swiglu_backward_saved_workspace_size()).  Same
 * reference caller as kda_swiglu_backward_bf16. */
size_t kda_swiglu_backward_saved_workspace_size(int64_t M, int64_t K, int64_t N);
kda_status kda_swiglu_backward_saved_bf16(const void* dout, const void* x, const void* w_up, const void* w_down,
                                          const void* w_gate, const void* g, const void* u, void* dx, void* dw_up,
                                          void* dw_down, void* dw_gate, int64_t M, int64_t K, int64_t N,
                                          void* workspace, size_t workspace_bytes, void* stream);

/* lora: out (M,N) = x @ w + (x @ a) @ b ; x (M,K), w (K,N), a (K,R), b (R,N).
 * The low-rank product t = x @ a (M,R) is kept in the workspace as bf16 and
 * accumulated into the same tensor-memory accumulator as x @ w; for R <= 128
 * the workspace also holds the fp32 partials of a K-split t = x @ a.
 * Replaces lora forward(x, w, a, b)
 * (workspaces/lora/runs/offline_lora_bf16_split_sim.py:175-180; kernel
 * workspaces/lora/runs/lora_v3_bf16_split.py:11). */
size_t kda_lora_workspace_size(int64_t M, int64_t K, int64_t N, int64_t R);
kda_status kda_lora_bf16(const void* x, const void* w, const void* a, const void* b, void* out, int64_t M,
                         int64_t K, int64_t N, int64_t R, void* workspace, size_t workspace_bytes, void* stream);

/* lora, fp32 in / out at fp32 accuracy: t = x @ a in fp32, then one
 * three-pass GEMM of [x | t] @ [w ; b] over K + R (the reference forward,
 * workspaces/lora/runs/offline_lora_bf16_split_sim.py:175-180, with its fp32 t).
 * R must be a multiple of 8. */
size_t kda_lora_f32_workspace_size(int64_t M, int64_t K, int64_t N, int64_t R);
kda_status kda_lora_f32(const float* x, const float* w, const float* a, const float* b, float* out, int64_t M,
                        int64_t K, int64_t N, int64_t R, void* workspace, size_t workspace_bytes, void* stream);

/* gqa_full: grouped-query attention, head_dim 128.
 * q (B,S,QH,128), k/v (B,S,KH,128) bf16 (row-major, [B,S,H,D]); query head
 * h reads kv head h / (QH/KH).  out = softmax(q k^T / sqrt(128) [+causal
 * mask]) v, fp32 softmax / accumulation, bf16 out.
 * rope_theta > 0 applies the half-split rotary embedding (angle =
 * pos * rope_theta^(-2i/128)) to q and k first; rope_theta <= 0 disables it.
 * out_bshd != 0 writes out as (B,S,QH,128); 0 writes the reference order
 * (B,QH,S,128).  The workspace (kda_gqa_full_workspace_size() bytes,
 * 16-byte aligned, always required) receives a transposed copy of v and, with
 * RoPE, the rotated q and k.
 * Replaces gqa_full forward(q, k, v)
 * (workspaces/gqa_full/runs/offline_score_bf16_split_sim.py:100-124; kernel
 * workspaces/gqa_full/runs/gqa_full_v7a_exp_from_psum.py:16). */
size_t kda_gqa_full_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, float rope_theta);
kda_status kda_gqa_full_bf16(const void* q, const void* k, const void* v, void* out, int64_t B, int64_t S,
                             int64_t QH, int64_t KH, int64_t D, int causal, float rope_theta, int out_bshd,
                             void* workspace, size_t workspace_bytes, void* stream);

/* gqa_full, fp32 q / k / v / out at fp32 accuracy, head by head: fp32 scores
 * from a three-pass split GEMM, a max-shifted fp32 row softmax (scale
 * 1/sqrt(D), optional causal mask) that writes the probabilities' split,
 * then P @ v_h.  Any D that is a multiple of 32; S a multiple of 8; no RoPE
 * (rope_theta must be <= 0).  The workspace holds the split q, k (transposed
 * per head), v and one head's scores and probabilities
 * (workspaces/gqa_full/runs/offline_score_bf16_split_sim.py:100-124). */
size_t kda_gqa_full_f32_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D);
kda_status kda_gqa_full_f32(const float* q, const float* k, const float* v, float* out, int64_t B, int64_t S,
                            int64_t QH, int64_t KH, int64_t D, int causal, float rope_theta, int out_bshd,
                            void* workspace, size_t workspace_bytes, void* stream);

/* gqa_full with the row statistics the backward needs: the same forward as
 * kda_gqa_full_bf16 (same workspace) that also writes lse [B][QH][S] fp32,
 * each query row's log2-sum-exp of the scaled scores (16-byte aligned).
 * The training-side forward of gqa_full forward(q, k, v)
 * (workspaces/gqa_full/runs/offline_score_bf16_split_sim.py:100-124); the
 * reference has no backward, so no counterpart for lse. */
kda_status kda_gqa_full_lse_bf16(const void* q, const void* k, const void* v, void* out, float* lse, int64_t B,
                                 int64_t S, int64_t QH, int64_t KH, int64_t D, int causal, float rope_theta,
                                 int out_bshd, void* workspace, size_t workspace_bytes, void* stream);

/* gqa_full backward: the gradients of gqa_full (head_dim 128) given
 * dout in the reference order (B,QH,S,128) bf16: dq (B,S,QH,128) and dk, dv
 * (B,S,KH,128), bf16.  The forward runs again first (its output and each
 * row's log2-sum-exp into the workspace); di = rowsum(dout * out); then one
 * flash-style kernel per (batch, kv head, 128-key block) walks the query
 * blocks with P and dS only in shared memory:
 *   P = 2^(q k^T log2e / sqrt(128) - lse) [causal: 0 for keys after the query];
 *   dS = P (dout v^T - di) ; dq = dS k / sqrt(128) ; dk = dS^T q / sqrt(128) ;
 *   dv = P^T dout
 * rope_theta > 0: the forward's RoPE -- the backward runs on the rotated q, k
 * (recomputed in the workspace) and rotates dq, dk back by the negated angle.
 * S a multiple of 8.  The training-side caller of gqa_full forward
 * (workspaces/gqa_full/runs/offline_score_bf16_split_sim.py:100-124); the
 * reference has no backward. */
size_t kda_gqa_full_backward_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                            float rope_theta);
kda_status kda_gqa_full_backward_bf16(const void* dout, const void* q, const void* k, const void* v, void* dq,
                                      void* dk, void* dv, int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                      int causal, float rope_theta, void* workspace, size_t workspace_bytes,
                                      void* stream);

/* gqa_full backward from a saved forward: as kda_gqa_full_backward_bf16, but
 * the forward's output `out` (reference order (B,QH,S,128) bf16, as written by
 * kda_gqa_full_lse_bf16 with out_bshd = 0) and its lse (B,QH,S fp32) are
 * passed in instead of recomputed -- the backward of a training step whose
 * forward kept them.  Smaller workspace (kda_gqa_full_backward_saved_
 * workspace_size()).  Same reference caller as kda_gqa_full_backward_bf16. */
size_t kda_gqa_full_backward_saved_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                                  float rope_theta);
kda_status kda_gqa_full_backward_saved_bf16(const void* dout, const void* q, const void* k, const void* v,
                                            const void* out, const float* lse, void* dq, void* dk, void* dv,
                                            int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, int causal,
                                            float rope_theta, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------- local attention --
 * The attention half of a decoder layer whose queries see a sliding window
 * and the sequence's first tokens.  No reference counterpart (the neighbours
 * of gqa_full).  Rows are head_dim contiguous values; *_strides are host
 * arrays of the element strides of the leading axes (batch, token, head), so
 * slices of a packed projection and layers of a cache are taken as they are:
 * every row must start on 16 bytes.  An axis of one entry may have any stride. */

/* rope_table: table [length][D/2][2] = cos, sin of position * theta^(-2 i / D)
 * (theta and the angles in double precision). */
kda_status kda_rope_table_f32(float* table, int64_t length, int64_t D, double theta, void* stream);

/* qk_norm_rope: for each head row x of q (B,S,QH,D) and k (B,S,KH,D),
 *   y = rotate(x / sqrt(mean x^2 + eps) * g, table[position])
 * (half-split rotation), written contiguous to q_out, k_out in the inputs'
 * type (bf16, or fp32 with f32 != 0); gq, gk (D,) fp32; D 64, 128 or 256.
 * positions: int32 [B][S], or NULL for 0 .. S-1.  A position outside
 * [0, table_len) gives NaN rows and sets 8 in the device error word. */
kda_status kda_qk_norm_rope(const void* q, const void* k, const float* gq, const float* gk, const float* table,
                            int64_t table_len, const int* positions, float eps, void* q_out, void* k_out, int64_t B,
                            int64_t S, int64_t QH, int64_t KH, int64_t D, const int64_t* q_strides,
                            const int64_t* k_strides, int f32, void* stream);

/* qk_norm_rope_append (bf16): the same for S new tokens of each request at
 * positions lengths[b] + s (int32 [B], tokens already cached): q_out (B,S,QH,D)
 * contiguous, the rotated k and v as it is into the caches (B,cache_len,KH,D,
 * strided) at those positions.  lengths[b] < 0: an idle slot, zeros and no
 * write.  A position outside the cache or the table: NaN, no write, 8 in
 * the device error word. */
kda_status kda_qk_norm_rope_append_bf16(const void* q, const void* k, const void* v, const float* gq,
                                        const float* gk, const float* table, int64_t table_len, const int* lengths,
                                        float eps, void* q_out, void* k_cache, void* v_cache, int64_t cache_len,
                                        int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                        const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                        const int64_t* k_cache_strides, const int64_t* v_cache_strides, void* stream);

/* Gradients of qk_norm_rope given those of its outputs (contiguous): dq, dk
 * contiguous in the inputs' type, dgq, dgk fp32 (D,), summed in a fixed order.
 * A position outside the table: NaN (its rows, dgq, dgk) and 8 in the device
 * error word. */
size_t kda_qk_norm_rope_backward_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D, int f32);
kda_status kda_qk_norm_rope_backward(const void* dq_out, const void* dk_out, const void* q, const void* k,
                                     const float* gq, const float* gk, const float* table, int64_t table_len,
                                     const int* positions, float eps, void* dq, void* dk, float* dgq, float* dgk,
                                     int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                     const int64_t* q_strides, const int64_t* k_strides, int f32, void* workspace,
                                     size_t workspace_bytes, void* stream);

/* gqa_window (bf16, D 128): causal attention in which query i sees key j <= i
 * where i - j < window or j < sinks; scores scaled by 1/sqrt(D).  out
 * (B,S,QH,D) contiguous; lse, if not NULL, [B][QH][S] fp32: each row's
 * log2-sum-exp of the scaled scores, for the backward.  No workspace. */
kda_status kda_gqa_window_bf16(const void* q, const void* k, const void* v, void* out, float* lse, int64_t B,
                               int64_t S, int64_t QH, int64_t KH, int64_t D, int64_t window, int64_t sinks,
                               const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                               void* stream);

/* Gradients of gqa_window given dout and the forward's out (B,S,QH,D,
 * contiguous) and lse: dq, dk, dv bf16, contiguous. */
size_t kda_gqa_window_backward_workspace_size(int64_t B, int64_t S, int64_t QH, int64_t KH, int64_t D,
                                              int64_t window, int64_t sinks);
kda_status kda_gqa_window_backward_bf16(const void* dout, const void* q, const void* k, const void* v,
                                        const void* out, const float* lse, void* dq, void* dk, void* dv, int64_t B,
                                        int64_t S, int64_t QH, int64_t KH, int64_t D, int64_t window, int64_t sinks,
                                        const int64_t* q_strides, const int64_t* k_strides,
                                        const int64_t* v_strides, void* workspace, size_t workspace_bytes,
                                        void* stream);

/* gqa_window_decode (bf16, D 128): gqa_window of the newest token of each
 * request, q (B,QH,D) (strides of batch and head), against the caches
 * (B,T,KH,D, strided) of which lengths[b] tokens are valid, the newest among
 * them; out (B,QH,D) contiguous.  lengths[b] <= 0: zeros; a length past T is
 * cut to T and sets 8 in the device error word.  No workspace. */
kda_status kda_gqa_window_decode_bf16(const void* q, const void* k_cache, const void* v_cache, const int* lengths,
                                      void* out, int64_t B, int64_t T, int64_t QH, int64_t KH, int64_t D,
                                      int64_t window, int64_t sinks, const int64_t* q_strides,
                                      const int64_t* k_strides, const int64_t* v_strides, void* stream);

/* ------------------------------------- packed sequences, 4-bit caches --
 * Attention over whole contexts: sequences of different lengths one behind
 * the other in one buffer of tokens, and a key/value cache held in 4 bits.  No
 * reference counterpart (the neighbours of gqa_full).  Rows and strides as
 * above; here *_strides have two entries, token and head, unless stated. */

/* packed_plan: the tables that gqa_packed and its backward work by, for
 * sequences s = rows [offsets[s], offsets[s+1]) of a buffer of `tokens` rows;
 * offsets: int32 [sequences+1] on the device, not falling, within [0, tokens]
 * (else: a plan of no sequences and 8 in the device error word).  One plan serves
 * every call on buffers of these offsets.  plan: 16-byte aligned, exactly the
 * size that the query returns. */
size_t kda_packed_plan_size(int64_t tokens, int64_t sequences);
kda_status kda_packed_plan(const int* offsets, int64_t sequences, int64_t tokens, void* plan, size_t plan_bytes,
                           void* stream);

/* gqa_packed (bf16, D 128): causal attention within each sequence, scores
 * scaled by 1/sqrt(D).  q (tokens,QH,D), k, v (tokens,KH,D); out
 * (tokens,QH,D) contiguous; lse, if not NULL, [QH][tokens] fp32: each row's
 * log2-sum-exp of the scaled scores, for the backward.  Rows of no sequence are
 * never read into a result; in out and lse they become zeros (zero_rest != 0)
 * or stay as they are.  A plan for another number of tokens: nothing is done
 * and 8 is set in the device error word.  A row's sums are divided at the end:
 * they have to stay within fp32, 2^8 |v| times the row's keys at most.  No
 * workspace. */
kda_status kda_gqa_packed_bf16(const void* q, const void* k, const void* v, const void* plan, size_t plan_bytes,
                               void* out, float* lse, int zero_rest, int64_t tokens, int64_t QH, int64_t KH,
                               int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, void* stream);

/* Gradients of gqa_packed given dout and the forward's out (tokens,QH,D,
 * contiguous) and lse: dq, dk, dv bf16, contiguous; rows of no sequence as in
 * the forward. */
size_t kda_gqa_packed_backward_workspace_size(int64_t tokens, size_t plan_bytes, int64_t QH, int64_t KH, int64_t D);
kda_status kda_gqa_packed_backward_bf16(const void* dout, const void* q, const void* k, const void* v,
                                        const void* out, const float* lse, const void* plan, size_t plan_bytes,
                                        void* dq, void* dk, void* dv, int zero_rest, int64_t tokens, int64_t QH,
                                        int64_t KH, int64_t D, const int64_t* q_strides, const int64_t* k_strides,
                                        const int64_t* v_strides, void* workspace, size_t workspace_bytes,
                                        void* stream);

/* The 4-bit cache: (B, KH, blocks, bytes of a block) uint8, for keys and for
 * values each, strided over request and head (byte strides, multiples of 16).
 * A block holds 16 tokens of one head: 16 rows of 64 bytes of codes, then
 * [16][128/group] pairs (step, low) of bf16; channel 32 g + 8 c + i of token t
 * is nibble i of the 32-bit word at byte 64 t + 16 (c ^ (t/2 & 3)) + 4 g, and
 * its value code * step + low with its group's pair.  group: 32, 64 or 128
 * channels.  All zeros is a valid cache.  q4_block_bytes: 1024 + 8192/group. */
size_t kda_q4_block_bytes(int64_t group);

/* kv_append_q4: new rows of k and v (bf16) into the caches, per group low =
 * min, step = bf16((max - low)/15), code = round((x - low)/step) (single fp32
 * operations, the quotient by step as a product with its fp32 reciprocal; a step
 * below 2^-126 becomes zero; a group that holds an infinity or a NaN, or whose
 * max - low is past fp32's largest number, reads back as NaN).
 * offsets NULL: tokens/B rows of each request, k and v (B,S,KH,D) with strides
 * of request, token and head; else int32 [B+1]: rows [offsets[b], offsets[b+1])
 * of k, v (tokens,KH,D) are request b's (strides[0] is not used), rows of none
 * are skipped.  Row i of request b goes to position lengths[b] + i (int32 [B]);
 * lengths[b] < 0: an idle slot, no write.  A position past the cache: no write
 * and 8 in the device error word. */
kda_status kda_kv_append_q4(const void* k, const void* v, const int* offsets, const int* lengths, void* k_cache,
                            void* v_cache, int64_t tokens, int64_t B, int64_t blocks, int64_t KH, int64_t D,
                            int64_t group, const int64_t* k_strides, const int64_t* v_strides,
                            const int64_t* k_cache_strides, const int64_t* v_cache_strides, void* stream);

/* kv_read_q4: every value of a cache, out (B, 16 blocks, KH, D) bf16. */
kda_status kda_kv_read_q4(const void* cache, void* out, int64_t B, int64_t blocks, int64_t KH, int64_t D,
                          int64_t group, const int64_t* cache_strides, void* stream);

/* gqa_decode_q4 (q, out bf16, D 128): gqa_window_decode against 4-bit caches.
 * A window of the cache's length or more sees all of it.  Finite values of any
 * size give the rounded sum, for up to 2^24 visible tokens; a product of weight
 * (relative to the largest) and value that is below 2^-94 loses bits.
 * |q| below 2^120.  Steps of the groups of a head (among the visible tokens) may
 * differ by 2^18 before the smaller ones' channels are off by more than bf16's rounding. */
size_t kda_gqa_decode_q4_workspace_size(int64_t QH, int64_t KH);
kda_status kda_gqa_decode_q4(const void* q, const void* k_cache, const void* v_cache, const int* lengths, void* out,
                             int64_t B, int64_t blocks, int64_t QH, int64_t KH, int64_t D, int64_t group,
                             int64_t window, int64_t sinks, const int64_t* q_strides,
                             const int64_t* k_cache_strides, const int64_t* v_cache_strides, void* workspace,
                             size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KDA_H_ */
