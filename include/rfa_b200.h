/*
 * rfa_b200 -- C ABI of the B200 (sm_100a) Random Feature Attention kernels.
 *
 * Plain pointers and sizes only; no framework types.  Every pointer is a DEVICE
 * pointer unless stated otherwise, every array is contiguous in the layout
 * given, and the caller owns all memory: the library never allocates or frees
 * (the one query function below tells the caller how much scratch to bring).
 * All launches are asynchronous on the stream handed in (a cudaStream_t passed
 * as void*; NULL = the legacy default stream) on the CURRENT device.
 *
 * Return value of every int function: 0 on success; a negative RFA_E* code for
 * a rejected argument (nothing was launched); a positive value is the
 * cudaError_t of a failed launch.  rfa_last_error() gives the text for the
 * calling thread's most recent failure.
 *
 * Upstream = Noahs-ARK/RFA, package random_feature_attention; "replaces" names
 * the upstream interface (file:line) each entry point stands in for.
 *
 * Shapes: T tokens (time-major), BH = batch*heads, K = 2*D = width of phi,
 * d = head_dim.  The tensor-core attention kernels are built for K == 128 and
 * d == 64 (the only geometry upstream's benchmarks and checks use).  Any other
 * K % 8 == 0, d % 8 == 0 whose fp32 state [K][d+1] fits in shared memory (e.g.
 * K <= 256 with d <= 128) runs in chunks of 16 to 64 tokens, state, weights and
 * sums in fp32 (an fp32 operand of a product as two parts of 11 bits and a sign),
 * where a chunk's tiles fit beside the state, else on
 * kernels that walk a sequence token by token, as upstream's do
 * (cuda/forward.cu:112-125); so do cross attention's query kernels and state
 * backward.
 * The packed-total / gathered-scan entry points of the sequence-sharded path and
 * rfa_causal_bwd_noalloc exist for K == 128, d == 64 only.  Unsupported
 * geometries are rejected with RFA_EUNSUPPORTED.  fp16 arrays are IEEE binary16.
 */
#ifndef RFA_B200_H_
#define RFA_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RFA_B200_VERSION 100

enum {
  RFA_OK = 0,
  RFA_EINVAL = -1,       /* null pointer, negative size, bad enum              */
  RFA_EALIGN = -2,       /* pointer not 16-byte aligned                        */
  RFA_EUNSUPPORTED = -3, /* geometry or dtype this build has no kernel for     */
  RFA_EWORKSPACE = -4,   /* workspace missing or too small                     */
  RFA_EDEVICE = -5       /* not an sm_100 device / driver entry point missing  */
};

/* element types accepted where a signature has a *_dtype argument (RFA_BF16 by the
 * state-space entry points at the end only) */
enum { RFA_F16 = 0, RFA_F32 = 1, RFA_BF16 = 2 };

typedef void* rfa_stream_t;

int rfa_version(void);
const char* rfa_last_error(void);

/* Device-side health of the tensor-core kernels on the current device.  Every wait
 * inside them is bounded (about four seconds of wall-clock time); a wait that runs out
 * records its site and the kernel leaves early (its outputs are then invalid).
 * rfa_debug_status(): 0 when no wait ever ran out, else 100 * kernel family + site code;
 * synchronises the device and clears the flag.
 * rfa_status_mirror_enable(): makes the kernels on the current device also write that
 * code to one word of mapped host memory (allocated once per process with cudaHostAlloc
 * by the first call; call it once per device, outside stream capture).
 * rfa_status_peek(): that word -- no synchronisation, no clearing -- so a host can look
 * after every call and learn of a failure in an EARLIER kernel without stalling.
 * No upstream counterpart (upstream never reads launch or device errors,
 * cuda/forward.cu:155). */
int rfa_debug_status(void);
int rfa_status_mirror_enable(void);
int rfa_status_peek(void);

/* ------------------------------------------------------------------------
 * Feature map  phi(x) = scale * [sin(W xhat) | cos(W xhat)], xhat = x/(|x|+1e-3)
 * replaces utils.py:100-120 (_normalize + random_project); W is the effective
 * matrix sigma*W/tau of utils.py:90-97, fp32 [H, D, d].
 * x [rows, H, d] (rows = T*B), phi [rows, H, 2D].  d <= 128, d % 8 == 0,
 * D % 8 == 0, D <= 128.
 * ---------------------------------------------------------------------- */
int rfa_feature_map_fwd(const void* x, int x_dtype, const float* w,
                        void* phi, int phi_dtype,
                        int64_t rows, int H, int d, int D, float scale,
                        rfa_stream_t stream);

/* Gradient of the above: g_x [rows,H,d] and g_w [H,D,d] fp32.  g_w is
 * ACCUMULATED into (atomic adds): the caller zeroes it.  g_w may be NULL. */
int rfa_feature_map_bwd(const void* x, int x_dtype, const float* w,
                        const void* g_phi, int g_dtype,
                        void* g_x, int gx_dtype, float* g_w,
                        int64_t rows, int H, int d, int D, float scale,
                        rfa_stream_t stream);

/* The same two with a row mask: row_mask [rows] bytes (may be NULL), non-zero =
 * the row's features are all zero and no gradient flows through it -- a padded
 * key.  replaces the separate masked_fill pass over phi_k in cuda_causal_rfa
 * (causal_attention.py:137-143) when the caller computes phi_k itself. */
int rfa_feature_map_fwd_masked(const void* x, int x_dtype, const float* w,
                               const uint8_t* row_mask, void* phi, int phi_dtype,
                               int64_t rows, int H, int d, int D, float scale,
                               rfa_stream_t stream);
int rfa_feature_map_bwd_masked(const void* x, int x_dtype, const float* w,
                               const uint8_t* row_mask, const void* g_phi, int g_dtype,
                               void* g_x, int gx_dtype, float* g_w,
                               int64_t rows, int H, int d, int D, float scale,
                               rfa_stream_t stream);

/* The same for two arrays of one shape that share w (q and k of a self-attention
 * layer: random_project is called on both, causal_attention.py:241-248) in ONE
 * launch: one ramp and one copy of W_h instead of two, and in the backward one g_w
 * accumulator for both (g_w receives the sum of the two contributions).  fp16
 * arrays with d = D = 64 only (RFA_EUNSUPPORTED otherwise); either mask may be
 * NULL. */
int rfa_feature_map_fwd_pair(const void* x_a, const void* x_b, const float* w,
                             const uint8_t* row_mask_a, const uint8_t* row_mask_b,
                             void* phi_a, void* phi_b,
                             int64_t rows, int H, int d, int D, float scale,
                             rfa_stream_t stream);
int rfa_feature_map_bwd_pair(const void* x_a, const void* x_b, const float* w,
                             const uint8_t* row_mask_a, const uint8_t* row_mask_b,
                             const void* g_phi_a, const void* g_phi_b,
                             void* g_x_a, void* g_x_b, float* g_w,
                             int64_t rows, int H, int d, int D, float scale,
                             rfa_stream_t stream);

/* Effective random matrices for a whole step in one launch:
 *   out[i] = sigma[i] * bank[idx[i]] * inv_tau[i],  i < n_out
 * bank [n_bank, D, d] (fp16 or fp32, resident on the device), idx [n_out] int64,
 * sigma [n_out, d] fp32 or NULL, inv_tau [n_out] fp32 or NULL, out [n_out, D, d]
 * fp32.  An index outside the bank sets *bad_index_flag (a device int the caller
 * zeroes) and yields zeros.  replaces the host-side gather of
 * sample_random_matrices (utils.py:62-87) plus build_random_matrices per layer
 * (utils.py:90-97). */
int rfa_gather_random_matrices(const void* bank, int bank_dtype, int64_t n_bank,
                               const int64_t* idx, int64_t n_out,
                               const float* sigma, const float* inv_tau, float* out,
                               int D, int d, int* bad_index_flag, rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * Causal RFA.  q,k [T,BH,K] fp16, v/out/g [T,BH,d] fp16, time-major.
 *   out_t = q_t^T S_t / max(q_t . z_t, 1),  S_t = S_in + sum_{s<=t} k_s v_s^T,
 *   z_t = z_in + sum_{s<=t} k_s.
 * replaces rfa_cuda.forward  (cuda/rfa_cuda.cpp:22-27 -> cuda/forward.cu:128-169)
 *      and rfa_cuda.backward (cuda/rfa_cuda.cpp:29-36 -> cuda/backward.cu:530-585),
 * reached from RFA.forward/backward (rfa.py:113-145).
 *
 * s_in/z_in ([BH,K,d] / [BH,K] fp32, may both be NULL = zeros) is the state of
 * tokens before this call's first token; s_out/z_out (may be NULL) receives
 * the state after its last token (prefill -> decode hand-off; segment carry).
 * workspace: rfa_causal_workspace_bytes(T,BH,K,d) bytes, 256-byte aligned.
 * rfa_causal_fwd needs none at K = 128, d = 64 below 1024 tokens or above 74
 * (batch, head) pairs (from 1024 tokens on with at most 74 it is RFA_EWORKSPACE);
 * other geometries may be given none (NULL, or one that does not fit) and then run
 * sequences whole, which costs time where few long ones leave the GPU idle.
 * ---------------------------------------------------------------------- */
size_t rfa_causal_workspace_bytes(int64_t T, int BH, int K, int d);

int rfa_causal_fwd(const void* q, const void* k, const void* v, void* out,
                   const float* s_in, const float* z_in,
                   float* s_out, float* z_out,
                   void* workspace, size_t workspace_bytes,
                   int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* Full backward.  ds_in/dz_in (NULL = zeros) is the reverse carry: the sum over
 * tokens AFTER this call's last token of q (x) grad_qs and of q*grad_qz. */
int rfa_causal_bwd(const void* q, const void* k, const void* v, const void* g,
                   void* gq, void* gk, void* gv,
                   const float* s_in, const float* z_in,
                   const float* ds_in, const float* dz_in,
                   void* workspace, size_t workspace_bytes,
                   int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* Backward without any caller scratch and without any allocation: the same two
 * sweeps as rfa_causal_bwd from a zero state (no carries), with the per-token
 * scalars kept in a fixed 4 MiB array inside the library (present on every GPU
 * that loads it).  For hosts that may not call cudaMalloc once they are running
 * (a server that owns all device memory in its own pools; a C caller without a
 * device allocator).  It has no counterpart in upstream, whose extension
 * allocates its outputs itself (cuda/backward.cu:556-558).
 *   - T * BH must not exceed rfa_causal_bwd_noalloc_max_token_heads() (524288);
 *     larger problems are refused with RFA_EWORKSPACE.
 *   - The first call on each device looks up the array's device address
 *     (cudaGetSymbolAddress), and a host thread's first launch of any kernel of
 *     this library binds the device's primary context to that thread
 *     (cudaSetDevice on the current device); make the first call on each device
 *     and from each calling thread before starting any stream capture.
 *   - All calls on a device share the one array: two calls whose kernels can
 *     overlap on the GPU (different streams, no dependency) race on it.  Calls
 *     on one stream are safe.  Nothing in it needs clearing between calls: each
 *     call's first sweep rewrites every element its second sweep reads.
 *   - Allocates nothing: no cudaMalloc, cudaFree, cudaHostAlloc or allocating
 *     library routine is called, on the first call or later. */
int64_t rfa_causal_bwd_noalloc_max_token_heads(void);
int rfa_causal_bwd_noalloc(const void* q, const void* k, const void* v, const void* g,
                           void* gq, void* gk, void* gv,
                           int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * Staged forms of the causal path: the same kernels, for callers that keep the
 * workspace (and the forward's output) from one call to the next -- an autograd
 * function between forward and backward, the shards of a split sequence between
 * their local steps and the exchange.  No counterpart upstream, whose backward
 * recomputes everything from (q, k, v) (rfa.py:126-145, cuda/backward.cu:303-371)
 * and whose kernels walk a whole sequence in one CTA (cuda/forward.cu:112-125).
 *
 * ws_has says what the workspace already holds FOR THESE SAME ARGUMENTS:
 *   RFA_WS_PARTIALS  per-segment sums of k (x) v and k, left by
 *                    rfa_causal_shard_total (the forward then skips that pass);
 *   RFA_WS_STATES    the states entering each segment, left by any forward call
 *                    with the same s_in/z_in (the backward then skips both the
 *                    pass and the scan);
 *   RFA_WS_DEN       the raw denominators q_t . z_t, left by a forward call with
 *                    save_den != 0.  Together with the forward's output `out`
 *                    the forward-direction sweep then recomputes neither the
 *                    scores nor the numerators and reads q only when a
 *                    reverse-state total is asked for or the sequence is cut
 *                    into segments.
 * A call that names something the workspace does not hold computes garbage.
 *
 * rfa_causal_shard_total: total_packed [BH, K*d + K] = [sum k (x) v | sum k] over
 * this call's tokens.  rfa_exclusive_scan_gathered: from gathered
 * [world, BH, K*d + K] (every shard's packed total, e.g. after an all-gather) the
 * sum over the shards before (reverse != 0: after) shard `rank`, as s_out
 * [BH,K,d] and z_out [BH,K].  rfa_causal_bwd_q_staged: as rfa_causal_bwd_q, with
 * the reverse-state total written packed (dtotal_packed, may be NULL) and `out`
 * (may be NULL without RFA_WS_DEN).  rfa_causal_bwd_saved: both sweeps.
 * ---------------------------------------------------------------------- */
enum { RFA_WS_EMPTY = 0, RFA_WS_PARTIALS = 1, RFA_WS_STATES = 2, RFA_WS_DEN = 4 };

int rfa_causal_fwd_staged(const void* q, const void* k, const void* v, void* out,
                          const float* s_in, const float* z_in,
                          float* s_out, float* z_out,
                          void* workspace, size_t workspace_bytes,
                          int64_t T, int BH, int K, int d,
                          int ws_has, int save_den, rfa_stream_t stream);
int rfa_causal_shard_total(const void* k, const void* v, float* total_packed,
                           void* workspace, size_t workspace_bytes,
                           int64_t T, int BH, int K, int d, rfa_stream_t stream);
int rfa_exclusive_scan_gathered(const float* gathered, int world, int rank, int reverse,
                                float* s_out, float* z_out,
                                int BH, int K, int d, rfa_stream_t stream);
int rfa_causal_bwd_q_staged(const void* q, const void* k, const void* v, const void* g,
                            const void* out, void* gq,
                            const float* s_in, const float* z_in, float* dtotal_packed,
                            void* workspace, size_t workspace_bytes,
                            int64_t T, int BH, int K, int d, int ws_has, rfa_stream_t stream);
int rfa_causal_bwd_saved(const void* q, const void* k, const void* v, const void* g,
                         const void* out, void* gq, void* gk, void* gv,
                         const float* s_in, const float* z_in,
                         const float* ds_in, const float* dz_in,
                         void* workspace, size_t workspace_bytes,
                         int64_t T, int BH, int K, int d, int ws_has, rfa_stream_t stream);

/* The two halves of the backward, for a sequence sharded across devices:
 * _bwd_q runs the forward-direction sweep (gq; leaves per-token scalars in the
 * workspace) and writes this shard's own reverse-state total to ds_seg/dz_seg;
 * after the shards have exchanged those, _bwd_kv runs the reverse sweep with
 * the carry ds_in/dz_in.  The same workspace must be passed to both. */
int rfa_causal_bwd_q(const void* q, const void* k, const void* v, const void* g,
                     void* gq, const float* s_in, const float* z_in,
                     float* ds_seg, float* dz_seg,
                     void* workspace, size_t workspace_bytes,
                     int64_t T, int BH, int K, int d, rfa_stream_t stream);
int rfa_causal_bwd_kv(const void* q, const void* k, const void* v, const void* g,
                      void* gk, void* gv, const float* ds_in, const float* dz_in,
                      void* workspace, size_t workspace_bytes,
                      int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * State reduction  s = sum_t k_t v_t^T [BH,K,d], z = sum_t k_t [BH,K]  (fp32)
 * over unpadded positions; k [T,BH,K], v [T,BH,d] fp16; pad_mask [B,T] bytes
 * (non-zero = padding, may be NULL), BH = B*H with bh = b*H + h.
 * replaces cross_attention.py:97-104 (masked_fill + einsum + sum); also the
 * per-shard total of the sequence-sharded causal path.
 * ---------------------------------------------------------------------- */
int rfa_cross_state_fwd(const void* phi_k, const void* v, const uint8_t* pad_mask,
                        float* s, float* z,
                        int64_t T, int B, int H, int K, int d, rfa_stream_t stream);

/* The same reduction over nseg contiguous runs of tokens at once (nseg CTAs per
 * (batch, head) instead of one, for few long sequences): s_part [BH,nseg,K,d],
 * z_part [BH,nseg,K] fp32, run i covering tokens [i*L, min(T,(i+1)*L)) with
 * L = rfa_state_partials_run_length(T, nseg) (a multiple of 128); the caller
 * sums over nseg.  No padding mask.  No counterpart upstream (its kernels walk a
 * whole sequence in one CTA, cuda/forward.cu:112-125); used for the per-shard
 * totals of the sequence-sharded causal path. */
int64_t rfa_state_partials_run_length(int64_t T, int nseg);
int rfa_state_partials(const void* phi_k, const void* v, float* s_part, float* z_part,
                       int64_t T, int BH, int K, int d, int nseg, rfa_stream_t stream);

/* Gradient of the reduction: g_phi_k [T,BH,K] (zero at padded rows),
 * g_v [T,BH,d] from d_s [BH,K,d], d_z [BH,K] fp32. */
int rfa_cross_state_bwd(const void* phi_k, const void* v, const uint8_t* pad_mask,
                        const float* d_s, const float* d_z,
                        void* g_phi_k, void* g_v,
                        int64_t T, int B, int H, int K, int d, rfa_stream_t stream);

/* out_t = phi_q_t . s / max(|phi_q_t . z|, 1);  phi_q [T,BH,K], out [T,BH,d] fp16.
 * replaces CrossAttention.rfa, cross_attention.py:266-269. */
int rfa_cross_query_fwd(const void* phi_q, const float* s, const float* z, void* out,
                        int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* Gradient of the above for upstream g [T,BH,d]: g_phi_q [T,BH,K] fp16 and the
 * state gradients d_s [BH,K,d], d_z [BH,K] fp32 (overwritten, not accumulated). */
int rfa_cross_query_bwd(const void* phi_q, const float* s, const float* z, const void* g,
                        void* g_phi_q, float* d_s, float* d_z,
                        int64_t T, int BH, int K, int d, rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * One incremental-decoding step, in place on the state:
 *   s += phi_k (x) v;  z += phi_k;  out = phi_q . s / max(phi_q . z, 1)
 * phi_q, phi_k [BH,K], v/out [BH,d] of in_dtype; s [BH,K,d], z [BH,K] of
 * state_dtype.  replaces the loop body of incremental_rfa,
 * causal_attention.py:42-50 (which allocates a new state every token).
 * ---------------------------------------------------------------------- */
int rfa_decode_step(const void* phi_q, const void* phi_k, const void* v, int in_dtype,
                    void* s, void* z, int state_dtype, void* out,
                    int BH, int K, int d, rfa_stream_t stream);

/* The same step from raw q,k [BH,d]: applies the feature map (W fp32 [H,D,d],
 * bh % H selects the head) inside the kernel.  K = 2*D. */
int rfa_decode_step_fused(const void* q, const void* k, const void* v, int in_dtype,
                          const float* w, float scale,
                          void* s, void* z, int state_dtype, void* out,
                          int BH, int H, int D, int d, rfa_stream_t stream);

/* Projections of n rows (a batch's one token each) by `count` (1 to 3) matrices
 * of one shape:  y[m] = x w[m]^T + b[m];  x [n, in], w[m] [out, in], b[m] [out]
 * (or NULL), y[m] [n, out] fp16, sums in fp32; in, out multiples of 8.  w, b, y
 * are HOST arrays of device pointers.
 * rm != NULL: the same launch forms the step's random matrices for
 * rfa_decode_step_fused,  w_eff [H, D, d] fp32 = (sigma * rm) * inv_tau from fp16
 * rm [H, D, d] and sigma [H, d] (or NULL), each product rounded to fp16.
 * replaces nn.Linear on one token and build_random_matrices,
 * causal_attention.py:222-248, utils.py:90-97. */
int rfa_linear_rows(const void* x, const void* const* w, const void* const* b,
                    void* const* y, int count, int n, int in, int out,
                    const void* rm, const void* sigma, float inv_tau, float* w_eff,
                    int H, int D, int d, rfa_stream_t stream);

/* The small parts of a layer's training step, fp16 with fp32 sums.
 * rfa_column_sums: out[m][c] = sum over rows of g[m][row][c] for `count` (1 to 3)
 * arrays [rows, cols], cols a multiple of 8 (bias gradients); g, out are HOST
 * arrays of device pointers.
 * rfa_layer_matrices: w_eff [H, D, d] fp32 = (sigma * rm) * inv_tau as in
 * rfa_linear_rows; pad_mask != NULL: row_mask [T, B] = pad_mask [B, T] transposed.
 * rfa_layer_matrices_bwd: from g_w [H, D, d] fp32, g_sigma [H, d] and / or
 * g_rm [H, D, d] (NULL: not wanted; sigma NULL: 1), d at most 256.
 * replace what autograd makes of nn.Linear and build_random_matrices,
 * causal_attention.py:222-248, utils.py:90-97. */
int rfa_column_sums(const void* const* g, void* const* out, int count, int64_t rows, int cols, rfa_stream_t stream);
int rfa_layer_matrices(const void* rm, const void* sigma, float inv_tau, float* w_eff, int H, int D, int d,
                       const uint8_t* pad_mask, uint8_t* row_mask, int64_t T, int B, rfa_stream_t stream);
int rfa_layer_matrices_bwd(const float* g_w, const void* rm, const void* sigma, float inv_tau, void* g_sigma, void* g_rm,
                           int H, int D, int d, rfa_stream_t stream);

/* One decoding step of cross attention for all L layers in one launch:
 *   out[l] = phi_q[l] . s_l / max(|phi_q[l] . z_l|, 1)
 * phi_q [L,BH,K], out [L,BH,d] of in_dtype; s_ptrs / z_ptrs: DEVICE arrays of L
 * pointers to the layers' fp32 states [BH,K,d] / [BH,K] (16-byte aligned; they do
 * not change while a sequence is decoded, so the arrays are built once).
 * replaces L calls of CrossAttention.rfa with tgt_len 1 (cross_attention.py:266-269). */
int rfa_cross_decode_step(const void* phi_q, int in_dtype,
                          const float* const* s_ptrs, const float* const* z_ptrs,
                          void* out, int L, int BH, int K, int d, rfa_stream_t stream);

/* Causal forward with the feature map inside the kernel: replaces
 * utils.random_project on q and k (utils.py:100-120, called at
 * causal_attention.py:241-248, with the masked_fill of padded keys at :137-143)
 * followed by RFA.forward (rfa.py:113-124, cuda/forward.cu:16-169).
 * x_q, x_k, v, out: [T, B*H, d] fp16, the head index fastest in the middle axis;
 * w [H, D, d] fp32 (the matrices build_random_matrices returns, sigma and 1/tau
 * folded in); row_mask [T, B] bytes, nonzero = padded key, or NULL; scale = the
 * feature scale (D^-1/2 upstream).  The features phi [T, B*H, 2D] are formed tile
 * by tile in shared memory and never written.  d = 64, D = 64 only.  One CTA per
 * (batch, head): meant for B*H of about the SM count or more.
 * s_in/z_in/s_out/z_out as in rfa_causal_fwd.  save_den != 0: the raw
 * denominators are left in `workspace` (rfa_causal_workspace_bytes(T, B*H, 2D, d))
 * where rfa_causal_bwd_saved(..., ws_has = RFA_WS_DEN) finds them, once the caller
 * has recomputed the features with rfa_feature_map_fwd[_masked]; otherwise the
 * workspace may be NULL. */
int rfa_causal_fwd_fused(const void* x_q, const void* x_k, const void* v,
                         const float* w, const uint8_t* row_mask, float scale,
                         void* out,
                         const float* s_in, const float* z_in,
                         float* s_out, float* z_out,
                         void* workspace, size_t workspace_bytes,
                         int64_t T, int B, int H, int d, int D,
                         int save_den, rfa_stream_t stream);

/* The same forward for a layer's evaluation pass, from what the layer holds: the
 * matrices as fp16 rm [H, D, d] with sigma [H, d] (or NULL) and 1 / tau, each
 * product rounded to fp16 as build_random_matrices does (utils.py:90-97), and the
 * padding mask as the layer gets it, pad_mask [B, T] bytes (or NULL).  No state
 * in or out, nothing kept for a backward. */
int rfa_causal_fwd_fused_layer(const void* x_q, const void* x_k, const void* v,
                               const void* rm, const void* sigma, float inv_tau,
                               const uint8_t* pad_mask, float scale, void* out,
                               int64_t T, int B, int H, int d, int D,
                               rfa_stream_t stream);

/* Measurement aid, no upstream counterpart: streams in [T, BH, 64*nb] fp16 through
 * shared memory with the tile pattern of the causal kernels (one CTA per (batch,
 * head), chunks of 128 tokens, nb boxes of 128 rows x 128 bytes per chunk, two
 * stages) and, with_store != 0, writes one [128][128] fp16 tile per chunk to out
 * [T, BH, 128].  No arithmetic: its time is the memory system's own for this
 * pattern; bench.py reports it beside the copy bandwidth. */
int rfa_stream_probe(const void* in, void* out, int64_t T, int BH, int nb, int with_store,
                     rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * State-space operators: the short causal convolution, the selective scan and
 * the gated group norm of a layer whose running state, like S and z above, has
 * one size whatever the sequence's length.  No upstream counterpart.
 *
 * Activations are time-major, [T, B, D] with D channels adjacent; an input may
 * have any other strides (in elements, *_t from token to token, *_b from batch
 * row to batch row), outputs and gradients are contiguous.  dtype (RFA_F16,
 * RFA_F32 or RFA_BF16) is the type of all activations; sums, states and their
 * gradients are fp32.  mask [B, T] bytes or NULL, non-zero = a padded token:
 * every result of the others is what it would be if padded tokens were not
 * there, whatever stands in them, and a padded token's outputs and gradients
 * are zero.  No alignment is asked for beyond the elements' own, except that
 * states, checkpoints and workspaces are 16-byte aligned.  T < 2^31 - 64,
 * B <= 65535, D and C <= 2^24 (convolution: T D < 2^44); a size of zero is
 * refused (there is nothing to launch).  Outputs overlap neither inputs nor each other,
 * but for states where that is said.  What a batch row holds reaches no other row's
 * results; the same call gives the same bits.
 * ---------------------------------------------------------------------- */

/* Causal depthwise convolution over the last W tokens (1 <= W <= 8):
 *   pre_t = bias + sum_j weight[.][j] x_(t - W + 1 + j),  y_t = silu(pre_t) or pre_t.
 * weight [D, W] and bias [D] (or NULL) of dtype.  state_in [B, W-1, D] of dtype, or
 * NULL for zeros: the inputs in front of the first token, oldest first; state_out, or
 * NULL: the last W - 1 inputs including those of state_in.  state_out may be state_in
 * where T is 1 (and not otherwise). */
typedef struct {
  const void* x;
  int64_t x_t, x_b;
  const void *weight, *bias, *state_in;
  const uint8_t* mask;
  int64_t T;
  int B, D, W, dtype, silu;
} rfa_causal_conv_t;
int rfa_causal_conv_fwd(const rfa_causal_conv_t* conv, void* y, void* state_out,
                        rfa_stream_t stream);
/* Gradients: g [T, B, D] with strides g_t, g_b, g_state [B, W-1, D] of the outgoing
 * state or NULL -> gx [T, B, D]; g_weight [D, W] and g_bias [D], g_state_in [B, W-1, D],
 * each or NULL. */
size_t rfa_causal_conv_workspace_bytes(int64_t T, int B, int D, int W);
int rfa_causal_conv_bwd(const rfa_causal_conv_t* conv, const void* g, int64_t g_t, int64_t g_b,
                        const void* g_state, void* gx, void* g_weight, void* g_bias, void* g_state_in,
                        void* workspace, size_t workspace_bytes, rfa_stream_t stream);

/* Selective scan, per batch row and channel i of group i / (D / G):
 *   delta_t = softplus(dt_t + dt_bias)     (dt_t + dt_bias where softplus is 0)
 *   s_t = exp(delta_t a) s_(t-1) + delta_t b_t x_t        (N states, 1 <= N <= 64)
 *   y_t = c_t . s_t + d x_t
 * x, dt [T, B, D]; b, c [T, B, G, N], the N adjacent, *_g from group to group; a [D, N]
 * (finite; delta a <= 88, or results are not defined), d [D] or NULL, dt_bias [D] or NULL,
 * states [B, D, N], all fp32. */
typedef struct {
  const void *x, *dt, *b, *c;
  int64_t x_t, x_b, dt_t, dt_b, b_t, b_b, b_g, c_t, c_b, c_g;
  const float *a, *d, *dt_bias, *s_in;      /* s_in NULL: zeros */
  const uint8_t* mask;
  int64_t T;
  int B, D, N, G, dtype, softplus;
} rfa_scan_t;
/* Scratch of a forward (backward = 0) or backward (1) call with `scan`'s sizes, and what
 * a forward leaves for the backward (the state in front of every 16th token, every 8th
 * with up to 8 states). */
size_t rfa_selective_scan_workspace_bytes(int64_t T, int B, int D, int N, int G, int backward);
size_t rfa_selective_scan_checkpoint_bytes(int64_t T, int B, int D, int N);
/* y [T, B, D]; s_out [B, D, N] or NULL (not s_in); checkpoints or NULL. */
int rfa_selective_scan_fwd(const rfa_scan_t* scan, void* y, float* s_out, float* checkpoints,
                           void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* g [T, B, D] contiguous, g_s [B, D, N] of the last state or NULL, the forward's
 * checkpoints -> gx, gdt [T, B, D], gb, gc [T, B, G, N] of dtype; ga [D, N]; gd, g_dt_bias
 * [D], gs_in [B, D, N], each or NULL. */
int rfa_selective_scan_bwd(const rfa_scan_t* scan, const void* g, const float* g_s,
                           const float* checkpoints, void* gx, void* gdt, float* ga, void* gb,
                           void* gc, float* gd, float* g_dt_bias, float* gs_in,
                           void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* One token (T = 1): the state s [B, D, N] is updated in place (s_in is not read). */
int rfa_selective_scan_step(const rfa_scan_t* scan, void* y, float* s, rfa_stream_t stream);

/* Group norm of rows: each of `groups` runs of C / groups (<= 16384) adjacent channels of
 * x's row is brought to mean 0 and variance 1 (eps added to the variance), times weight
 * plus bias ([C] of dtype, each or NULL): n.  y = n silu(gate) with a gate, else silu(n);
 * n gate and n where silu is 0.  x, gate rows x_r, gate_r elements apart; y [rows, C]. */
typedef struct {
  const void* x;
  const void* gate;
  int64_t x_r, gate_r;
  const void *weight, *bias;
  int64_t rows;
  int C, groups, dtype, silu;
  float eps;
} rfa_group_norm_t;
int rfa_group_norm_fwd(const rfa_group_norm_t* norm, void* y, rfa_stream_t stream);
/* g rows g_r elements apart -> gx [rows, C]; g_gate [rows, C], g_weight, g_bias [C], each
 * or NULL. */
size_t rfa_group_norm_workspace_bytes(int64_t rows, int C, int groups);
int rfa_group_norm_bwd(const rfa_group_norm_t* norm, const void* g, int64_t g_r, void* gx,
                       void* g_gate, void* g_weight, void* g_bias,
                       void* workspace, size_t workspace_bytes, rfa_stream_t stream);

/* ------------------------------------------------------------------------
 * Attention of bounded memory beside causal RFA: linear attention whose state
 * decays, and softmax attention over a sliding window.  No upstream counterpart.
 *
 * Activations are time-major, [T, B, H, width] with a head's numbers adjacent; an
 * input may have any other strides (in elements: *_t from token to token, *_b from
 * batch row to batch row, *_h from head to head), outputs and gradients are
 * contiguous.  dtype (RFA_F16, RFA_F32 or RFA_BF16) is the type of all activations;
 * states, sums and softmax statistics are fp32.  mask [B, T] bytes or NULL, non-zero
 * = a padded token: every result of the others is what it would be if padded tokens
 * were not there, whatever stands in them, and a padded token's outputs and
 * gradients are zero.  States, caches, outputs and workspaces are 16-byte aligned, else
 * no alignment is asked for.  Heads of at most 256; T < 2^31 - 256, B and H <= 65535,
 * B H < 2^24; a size of zero is refused.  Outputs overlap neither inputs nor each
 * other, but for states and caches where that is said.  What a batch row holds reaches
 * no other row's results; the same call gives the same bits.
 * ---------------------------------------------------------------------- */

/* Linear attention with a decay for each head:
 *   S_t = e^(log_decay_t) S_(t-1) + k_t (x) v_t,   out_t = scale q_t S_t
 * q, k [T, B, H, K], v and out [T, B, H, D], states [B, H, K, D] fp32 (s_in NULL:
 * zeros), log_decay of decay_dtype with strides g_*, zero where it does not depend on
 * the token or the batch row. */
typedef struct {
  const void *q, *k, *v;
  int64_t q_t, q_b, q_h, k_t, k_b, k_h, v_t, v_b, v_h;
  const void* log_decay;
  int64_t g_t, g_b, g_h;
  const float* s_in;
  const uint8_t* mask;
  int64_t T;
  int B, H, K, D, dtype, decay_dtype;
  int per_head;              /* backward: g_decay is [H], the sum over tokens and batch rows; else [T, B, H] */
  float scale;
} rfa_decay_t;
size_t rfa_decay_workspace_bytes(int64_t T, int B, int H, int K, int D, int dtype, int backward);
/* s_out: the last state, or NULL; it may be s_in.  kept: rfa_decay_kept_bytes(decay) bytes
 * that a backward with the same `decay` goes on from, or NULL. */
size_t rfa_decay_kept_bytes(const rfa_decay_t* decay);
int rfa_decay_fwd(const rfa_decay_t* decay, void* out, float* s_out, void* kept,
                  void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* g [T, B, H, D] contiguous, g_s [B, H, K, D] of the last state or NULL, the forward's
 * kept or NULL (it is then computed again) -> gq, gk, gv; g_decay of decay_dtype and gs_in
 * [B, H, K, D], each or NULL. */
int rfa_decay_bwd(const rfa_decay_t* decay, const void* g, const float* g_s, const void* kept, void* gq,
                  void* gk, void* gv, void* g_decay, float* gs_in,
                  void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* One token (T = 1): the state s is updated in place (s_in is not read). */
int rfa_decay_step(const rfa_decay_t* decay, void* out, float* s, rfa_stream_t stream);

/* Softmax attention over a sliding window: token i sees token j <= i where i - j <
 * window or j < sinks (the first tokens stay visible), padded tokens not counted.
 *   out_i = sum_j softmax_j(scale q_i . k_j) v_j
 * q and out [T, B, H, D], k, v [T, B, G, D]; query heads h G / H ... share a key head.
 * A query that is padded gets zero. */
typedef struct {
  const void *q, *k, *v;
  int64_t q_t, q_b, q_h, k_t, k_b, k_h, v_t, v_b, v_h;
  const uint8_t* mask;
  int64_t T;
  int B, H, G, D, dtype, window, sinks;
  float scale;
} rfa_window_t;
/* Scratch of a forward (backward = 0) or backward (1) call. */
size_t rfa_window_workspace_bytes(int64_t T, int B, int H, int G, int D, int dtype, int window, int sinks, int backward);
/* lse [B, H, T] fp32, or NULL: what the backward wants of the softmax. */
int rfa_window_fwd(const rfa_window_t* window, void* out, float* lse,
                   void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* g, out [T, B, H, D] contiguous -> gq [T, B, H, D], gk, gv [T, B, G, D]. */
int rfa_window_bwd(const rfa_window_t* window, const void* out, const float* lse,
                   const void* g, void* gq, void* gk, void* gv,
                   void* workspace, size_t workspace_bytes, rfa_stream_t stream);
/* Decoding.  The cache: cache_k, cache_v [B, G, sinks + window, D] of dtype, length [B]
 * int64, the number of tokens so far (below 2^40).  Token number p is kept at p where p <
 * sinks, else at sinks + (p - sinks) % window.  The call appends its T tokens, attends
 * and updates cache and length in place; empty != 0: nothing is in the cache yet,
 * whatever length holds.  Slots that hold no token are neither read nor written. */
size_t rfa_window_append_workspace_bytes(int64_t T, int B, int H, int G, int D, int dtype, int window, int sinks, int empty);
int rfa_window_append(const rfa_window_t* window, void* cache_k, void* cache_v, int64_t* length, int empty,
                      void* out, void* workspace, size_t workspace_bytes, rfa_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* RFA_B200_H_ */
