/*
 * jakal_b200.h — C ABI of the B200-native (sm_100a) Jakal-Net operator hot path.
 *
 * Every entry point takes raw device pointers, sizes, dtype codes and a CUDA stream,
 * launches asynchronously on that stream and returns an int status (JK_OK == 0, negative
 * codes below). No entry point allocates device memory except where stated; callers own
 * every buffer. Inputs are read-only and C-contiguous; outputs are fully overwritten.
 *
 * Reference interfaces (Ahnd6474/Jakal-Net, paths relative to that project) that each
 * entry point replaces are cited beside the declaration.
 */
#ifndef JAKAL_B200_H_
#define JAKAL_B200_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (jk_status_string gives the text) ---------------------------------- */
#define JK_OK 0
#define JK_ERR_BAD_SHAPE (-1)          /* sizes inconsistent or out of the supported range */
#define JK_ERR_BAD_DTYPE (-2)          /* dtype code unknown or not supported by this op  */
#define JK_ERR_UNSUPPORTED_KIND (-3)   /* compress / scorer kind not implemented          */
#define JK_ERR_UNSUPPORTED_DEVICE (-4) /* no sm_100 device, or pointer not on the device  */
#define JK_ERR_LAUNCH (-5)             /* CUDA launch / runtime error                     */
#define JK_ERR_DEVICE_TIMEOUT (-6)     /* a bounded device-side wait gave up              */
#define JK_ERR_BAD_ARG (-7)            /* null pointer, negative k, bad window, ...       */
#define JK_ERR_ALIGNMENT (-8)          /* pointer not 16-byte aligned where required      */

/* ---- dtype codes --------------------------------------------------------------------- */
#define JK_F32 0
#define JK_BF16 1
#define JK_F16 2
/* Projection planes only: f32 projections (rank <= 32) stored as three bf16 planes
 * [h | m | l | 0] of 32 columns each (rp = 128), see jk_split3_bf16; the score tiles then
 * sum the six cross products, which reproduces an f32 dot product. */
#define JK_BF16X3 3

/* ---- edge / route compressors --------------------------------------------------------- */
#define JK_SOFTSIGN 0              /* s / (1 + |s|)                       propagation.py:85   */
#define JK_SIGNED_ABS_SOFTMAX 1    /* sign(s) * softmax(|s|)              propagation.py:74-82 */
#define JK_SIGNED_ENTMAX15 2       /* sign(s) * entmax15(|s|)             kernels.py:155-236  */
#define JK_SOFTMAX 3               /* softmax(s)  (routes)                transition.py:187-194 */

/* ---- multi-head scorers (MultiHeadPairwise / MultiHeadRoute, modules.py:259-302) ------ */
#define JK_HEADS_MAX 0              /* max_h s_h                       modules.py:291-298   */
#define JK_HEADS_SMOOTHMAX 1        /* logsumexp_h s_h - log H         modules.py:276-280   */
#define JK_HEADS_SIGNED_SMOOTHMAX 2 /* sum_h s_h * softmax_h(|s_h|)    modules.py:281-284   */

/* Multi-head scorer for the *_mh entry points. The projection rows hold `heads` blocks of
 * 16 * kph columns (head h at columns [16 kph h, 16 kph (h + 1)), zero padded up to rp);
 * the score of head h is the f32 dot of its blocks plus head_bias[h], and the heads are
 * combined per pair by `combine` before selection / compression. Replaces the
 * multihead_{max,smoothmax,signed_smoothmax}_low_rank_bilinear pairwise kinds and the
 * multihead_max_low_rank_bilinear_route (kernel_common.py:151-178;
 * jakal_net_native.cpp:724-776; jakal_net_native_cuda.cu:881-1027, 1186-1350). */
typedef struct jk_heads {
  int heads;              /* 2..4 (top-k kernels), 2 (window / dense kernels)        */
  int kph;                /* 16-column K steps per head; heads * 16 * kph <= rp       */
  int combine;            /* JK_HEADS_*                                              */
  const float* head_bias; /* device, `heads` floats added before combining, or NULL  */
} jk_heads_t;

typedef struct CUstream_st* jk_stream_t; /* == cudaStream_t; NULL = legacy default stream */

/* Human-readable text for a status code. */
const char* jk_status_string(int status);

/* Library / device probe. Returns JK_OK when the current device is sm_100 and the
 * kernels can launch; otherwise JK_ERR_UNSUPPORTED_DEVICE. Replaces the loader probes
 * native_backend.py:98-178 (supported_devices) / jakal_net_native.cpp:5914-5931. */
int jk_device_check(void);

/* Synchronises `stream`, then reads and clears the library's device-side error word
 * (set by a kernel whose bounded wait gave up). *device_status receives JK_OK or
 * JK_ERR_DEVICE_TIMEOUT. */
int jk_device_status(jk_stream_t stream, int* device_status);

/* Padded projection width the fused kernels expect for a score rank `rank`
 * (rank rounded up to a multiple of 64). */
int64_t jk_padded_rank(int64_t rank);

/*
 * Low-rank projection prologue (tcgen05 GEMM):
 *   out[r, c] = round(x[r, :] . w[c, :])                         c <  rank
 *   then, if core != NULL:  out = round(out * core[c])
 *   then, if temperature != 1: out = round(out / temperature)
 *   out[r, c] = 0 for rank <= c < out_stride (padding)
 * x [rows, dim], w [rank, dim], core [rank], out [rows, out_stride]; all in `dtype`
 * (JK_BF16 or JK_F16); round() = round-to-nearest into dtype, matching a torch.matmul in
 * the input dtype followed by the elementwise ops in that dtype.
 * Requirements: dim % 8 == 0, rank <= 128, out_stride == jk_padded_rank(rank).
 * Replaces the projection steps of jakal_net_native.cpp:6236-6239 (propagation) and
 * :6977-6986 (pairwise-route transition); native_backend.py:4445-4458.
 */
int jk_lowrank_project(const void* x, int64_t rows, int64_t dim, const void* w, int64_t rank,
                       const void* core, float temperature, int dtype, void* out,
                       int64_t out_stride, jk_stream_t stream);

/* The target and source projections of a propagation in one pass over x (rank <= 64,
 * bf16 / f16): out = round(x . w^T) and out2 = round(round(x . w2^T) * core) [/ T], each
 * [rows, 64]; one N = 128 GEMM against w and w2 stacked. Replaces the two matmuls of
 * jakal_net_native.cpp:6236-6239 (same rounding points as jk_lowrank_project). */
int jk_lowrank_project_pair(const void* x, int64_t rows, int64_t dim, const void* w, const void* w2,
                            int64_t rank, const void* core, float temperature, int dtype, void* out,
                            void* out2, jk_stream_t stream);

/*
 * Fused per-row top-k aggregate (tcgen05 score GEMM + streaming top-k + gather):
 *   score[b,t,s] = row_proj[b,t,:] . col_proj[b,s,:]              (f32 accumulation)
 *   visible(t,s) = s < n_cols and (window < 0 or t - window <= s <= t)
 *   sel(t)       = the min(k, #visible) visible s with the largest score, ties to the
 *                  lower s
 *   e[t,s]       = compress(score + score_bias) over sel(t)        (compress = JK_*)
 *   w[t,s]       = e[t,s] * (col_sender ? col_sender[b,s] : 1)
 *   out_state[b,t]  = sum_{s in sel(t)} w[t,s] * col_state[b,s]
 *   out_val[b,t,:]  = sum_{s in sel(t)} w[t,s] * col_val[b,s,:]
 * score_bias is added to every score; when bias_dev != NULL the f32 it points to (device
 * memory) is added as well, so a bias tensor needs no host synchronisation.
 * Shapes: row_proj [B, n_rows, rp], col_proj [B, n_cols, rp] (rp = jk_padded_rank, dtype
 * proj_dtype = JK_BF16 | JK_F16 | JK_BF16X3); col_state and col_sender [B, n_cols] in state_dtype;
 * col_val [B, n_cols, dim] in val_dtype; out_state [B, n_rows], out_val [B, n_rows, dim] in
 * out_dtype. Optional out_scores f32 [B, n_rows, k] (score + bias, sorted descending,
 * -inf in empty slots) and out_index int64 [B, n_rows, k] (-1 in empty slots).
 * 1 <= k <= 64. rp <= 128.
 * Replaces low_rank_propagation_topk_forward_cuda (jakal_net_native_cuda.cu:2545-2660,
 * kernel :1029-1183) as called from propagation_topk (jakal_net_native.cpp:6355-6389);
 * the window > 0 form is the window-intersect-top-k operator built from
 * kernel_common.py:433-456 + propagation.py:67-88.
 */
int jk_propagation_topk_forward(const void* row_proj, const void* col_proj, int64_t batch,
                                int64_t n_rows, int64_t n_cols, int64_t rp, int proj_dtype,
                                const void* col_state, const void* col_sender, int state_dtype,
                                const void* col_val, int64_t dim, int val_dtype, int64_t k,
                                int64_t window, float score_bias, const float* bias_dev,
                                int compress, void* out_state, void* out_val, int out_dtype,
                                float* out_scores, int64_t* out_index, jk_stream_t stream);

/*
 * Fused window / dense propagation without top-k (flash-style: tcgen05 score tile -> exact
 * f32 edges -> bf16 hi + lo edge tiles -> tcgen05 value GEMM, TMEM accumulator):
 *   visible(t,s) = s < n_cols and (window < 0 or t - window <= s <= t)
 *   e[t,s]       = compress over the visible s of row t of (score + score_bias (+ *bias_dev))
 *                  compress = JK_SOFTSIGN | JK_SIGNED_ABS_SOFTMAX | JK_SIGNED_ENTMAX15
 *   out_state[b,t] = sum_s e * col_state[b,s],  out_val[b,t,:] = sum_s e * col_val[b,s,:]
 * row_proj [B,n_rows,rp], col_proj [B,n_cols,rp] (JK_BF16 | JK_F16 | JK_BF16X3); col_val
 * [B,n_cols,dim] in the projections' 16-bit type (bf16 for JK_BF16X3), dim % 64 == 0; for
 * f32 values pass the bf16 hi plane as col_val and the lo plane as col_val_lo (see
 * jk_split2_bf16), else col_val_lo = NULL. col_state in state_dtype; outputs in out_dtype.
 * Replaces propagation_window / propagation_dense / propagation_query_dense
 * (jakal_net_native.cpp:6190-6303, 5962-6076, 6078-6188) and the CUDA kernels
 * jakal_net_native_cuda.cu:1579-1750, 2023-2109, 1388-1576.
 */
int jk_propagation_window_forward(const void* row_proj, const void* col_proj, int64_t batch,
                                  int64_t n_rows, int64_t n_cols, int64_t rp, int proj_dtype,
                                  const void* col_state, int state_dtype, const void* col_val,
                                  const void* col_val_lo, int64_t dim, int64_t window,
                                  float score_bias, const float* bias_dev, int compress,
                                  void* out_state, void* out_val, int out_dtype,
                                  jk_stream_t stream);

/* Dense pairwise transition (Transition.forward with a dense route, transition.py:238-254):
 * every source routes to every destination, routes compressed over the destinations of
 * the source (JK_SOFTMAX | JK_SIGNED_ABS_SOFTMAX | JK_SIGNED_ENTMAX15), times the source's
 * sender strength, accumulated into the destinations:
 *   out_state[d] = sum_s r[s,d] * sender[s] * src_state[s],
 *   out_val[d]   = sum_s r[s,d] * sender[s] * src_val[s].
 * src_proj [B, n_src, rp] (route source projection divided by the temperature) and
 * dst_proj [B, n_dst, rp]; logits = src_proj . dst_proj + score_bias (+ *bias_dev).
 * stats: caller scratch of batch * n_src * 3 floats (per-source max, sender / normaliser,
 * entmax threshold). dim % 64 == 0; f32 values as bf16 hi (src_val) + lo (src_val_lo)
 * planes, like jk_propagation_window_forward.
 * Replaces transition_pairwise_dense (jakal_net_native.cpp:6705-6914; native_backend.py
 * :5801-5822). */
int jk_transition_pairwise_dense_forward(const void* src_proj, const void* dst_proj, int64_t batch,
                                         int64_t n_src, int64_t n_dst, int64_t rp, int proj_dtype,
                                         const void* src_state, const void* sender, int state_dtype,
                                         const void* src_val, const void* src_val_lo, int64_t dim,
                                         float score_bias, const float* bias_dev, int compress,
                                         float* stats, void* out_state, void* out_val, int out_dtype,
                                         jk_stream_t stream);

/* Row block of a propagation / per-query top-k (row-sharded multi-GPU): the arguments of
 * jk_propagation_topk_forward over the FULL tensors, computing only the rows
 * [row_begin, row_begin + row_count) (row_begin a multiple of 128; row_count a multiple of
 * 128 unless the block runs to the last row); the other output rows are not written.
 * Nothing in the reference corresponds (its kernels run on one GPU); this is the per-rank
 * step of the query-row-block partition, whose outputs an all-gather then assembles. */
int jk_propagation_topk_rows_forward(const void* row_proj, const void* col_proj, int64_t batch,
                                     int64_t n_rows, int64_t row_begin, int64_t row_count,
                                     int64_t n_cols, int64_t rp, int proj_dtype, const void* col_state,
                                     const void* col_sender, int state_dtype, const void* col_val,
                                     int64_t dim, int val_dtype, int64_t k, int64_t window,
                                     float score_bias, const float* bias_dev, int compress,
                                     void* out_state, void* out_val, int out_dtype, float* out_scores,
                                     int64_t* out_index, jk_stream_t stream);

/* Multi-head variants: the entry point of the same name without _mh, with the scorer
 * `heads` (jk_heads_t above; 16-bit projections only, not JK_BF16X3). */
int jk_propagation_topk_forward_mh(const void* row_proj, const void* col_proj, int64_t batch,
                                   int64_t n_rows, int64_t n_cols, int64_t rp, int proj_dtype,
                                   const void* col_state, const void* col_sender, int state_dtype,
                                   const void* col_val, int64_t dim, int val_dtype, int64_t k,
                                   int64_t window, float score_bias, const float* bias_dev,
                                   int compress, void* out_state, void* out_val, int out_dtype,
                                   float* out_scores, int64_t* out_index, const jk_heads_t* heads,
                                   jk_stream_t stream);
int jk_transition_query_topk_forward_mh(const void* query_proj, const void* source_proj, int64_t batch,
                                        int64_t n_query, int64_t n_source, int64_t rp, int proj_dtype,
                                        const void* source_state, const void* source_sender,
                                        int state_dtype, const void* source_val, int64_t dim,
                                        int val_dtype, int64_t k, float score_bias,
                                        const float* bias_dev, int compress, void* out_state,
                                        void* out_val, int out_dtype, float* out_scores,
                                        int64_t* out_index, const jk_heads_t* heads, jk_stream_t stream);
int jk_transition_pairwise_topk_forward_mh(const void* src_proj, const void* dst_proj, int64_t batch,
                                           int64_t n_src, int64_t n_dst, int64_t rp, int proj_dtype,
                                           const void* src_state, const void* src_sender, int state_dtype,
                                           const void* src_val, int64_t dim, int val_dtype, int64_t k,
                                           float score_bias, const float* bias_dev, int compress,
                                           float* accum, void* out_state, void* out_val, int out_dtype,
                                           const jk_heads_t* heads, jk_stream_t stream);
int jk_propagation_window_forward_mh(const void* row_proj, const void* col_proj, int64_t batch,
                                     int64_t n_rows, int64_t n_cols, int64_t rp, int proj_dtype,
                                     const void* col_state, int state_dtype, const void* col_val,
                                     const void* col_val_lo, int64_t dim, int64_t window,
                                     float score_bias, const float* bias_dev, int compress,
                                     void* out_state, void* out_val, int out_dtype,
                                     const jk_heads_t* heads, jk_stream_t stream);
int jk_transition_pairwise_dense_forward_mh(const void* src_proj, const void* dst_proj, int64_t batch,
                                            int64_t n_src, int64_t n_dst, int64_t rp, int proj_dtype,
                                            const void* src_state, const void* sender, int state_dtype,
                                            const void* src_val, const void* src_val_lo, int64_t dim,
                                            float score_bias, const float* bias_dev, int compress,
                                            float* stats, void* out_state, void* out_val, int out_dtype,
                                            const jk_heads_t* heads, jk_stream_t stream);

/* f32 -> three bf16 planes [h|m|l|0] of 32 columns (rank <= 32), out [rows, 128] bf16, for
 * JK_BF16X3 projections. Replaces nothing: the reference computes these dots in f32. */
int jk_split3_bf16(const float* x, int64_t rows, int64_t rank, void* out, jk_stream_t stream);

/* f32 -> bf16 hi plane + bf16 lo plane (x - hi), n elements each, for f32 values. */
int jk_split2_bf16(const float* x, int64_t n, void* hi, void* lo, jk_stream_t stream);

/* f32 x [batch, rows, cols] (plus, when extra_col is not NULL, extra_col [batch, rows] as
 * column cols) -> bf16 out [batch, nblk * rows, out_cols]: block k (rows [k * rows,
 * (k + 1) * rows) of every batch item) holds the hi plane bf16(x) when bit k of plane_bits is
 * 0, the lo plane bf16(x - hi) when it is 1; columns past the data are zero. Stacking the
 * route matrix as (hi, hi, lo) and the values as (hi, lo, hi) makes one GEMM over the stacked
 * dimension sum the three products of an f32-accurate split GEMM. nblk <= 4. Replaces
 * nothing in the reference (its scatter adds f32 routes into f32 accumulators). */
int jk_split_stack_bf16(const float* x, const float* extra_col, int64_t batch, int64_t rows, int64_t cols,
                        int64_t out_cols, int nblk, unsigned plane_bits, void* out, jk_stream_t stream);

/*
 * Per-query ("query top-k") transition: identical contract to
 * jk_propagation_topk_forward with rows = query slots (row_proj = target-side route
 * projection of query_val), columns = source nodes (col_proj = core-weighted,
 * temperature-scaled source projection), compress = JK_SOFTMAX and
 * col_sender = sender strength softplus(src.state); window must be -1.
 * Replaces transition_query_topk (jakal_net_native.cpp:7089-7246) and
 * query_topk_reduce_cuda (jakal_net_native_cuda.cu:2335-2417).
 */
int jk_transition_query_topk_forward(const void* query_proj, const void* source_proj,
                                     int64_t batch, int64_t n_query, int64_t n_source,
                                     int64_t rp, int proj_dtype, const void* source_state,
                                     const void* source_sender, int state_dtype,
                                     const void* source_val, int64_t dim, int val_dtype,
                                     int64_t k, float score_bias, const float* bias_dev,
                                     int compress, void* out_state, void* out_val,
                                     int out_dtype, float* out_scores, int64_t* out_index,
                                     jk_stream_t stream);

/*
 * Per-source sparse transition (SparseTransition):
 *   logit[b,i,j] = src_proj[b,i,:] . dst_proj[b,j,:] + score_bias (+ *bias_dev)
 *                  (src_proj already core-weighted and temperature-scaled)
 *   sel(i)       = top-k destinations j of source i, ties to the lower j
 *   r[i,j]       = compress(logit) over sel(i)        (JK_SOFTMAX / SIGNED_ABS / ENTMAX15)
 *   out_state[b,j] = sum_i r[i,j] * src_sender[b,i] * src_state[b,i]
 *   out_val[b,j,:] = sum_i r[i,j] * src_sender[b,i] * src_val[b,i,:]
 * src_state / src_sender in state_dtype, src_val in val_dtype. `accum` is caller-provided
 * f32 scratch of B*n_dst*(dim+1) elements, 16-byte aligned (zeroed by the call); outputs
 * are written in out_dtype. 1 <= k <= 64.
 * Replaces low_rank_pairwise_topk_forward_cuda (jakal_net_native_cuda.cu:2420-2542,
 * kernel :740-878) as called from transition_pairwise_topk
 * (jakal_net_native.cpp:6958-7007).
 */
int jk_transition_pairwise_topk_forward(const void* src_proj, const void* dst_proj,
                                        int64_t batch, int64_t n_src, int64_t n_dst,
                                        int64_t rp, int proj_dtype, const void* src_state,
                                        const void* src_sender, int state_dtype,
                                        const void* src_val, int64_t dim, int val_dtype,
                                        int64_t k, float score_bias, const float* bias_dev,
                                        int compress, float* accum, void* out_state,
                                        void* out_val, int out_dtype, jk_stream_t stream);

/*
 * Routes form of the per-source sparse transition (deterministic, no atomics):
 *   routes[b, s, d] = compress(logit[b, s, :] over sel(s))[d] * (src_sender ? src_sender[b, s] : 1)
 * for the k selected destinations d of every source s (selection, bias and compressors as
 * jk_transition_pairwise_topk_forward); every other entry is left untouched, so the caller
 * zeroes routes (f32 [B, n_src, n_dst]) first. The aggregate
 *   out_state[b, d] = sum_s routes[b, s, d] * src_state[b, s],
 *   out_val[b, d, :] = sum_s routes[b, s, d] * src_val[b, s, :]
 * is then a plain GEMM (routes^T x values), with no atomics and a fixed summation order.
 * Optional out_scores f32 / out_index int64 [B, n_src, k]: every source's selection (logit +
 * bias, in descending order, -inf / -1 in empty slots) -- what the backward of the route
 * scores needs (native_backend.py:4459-4491).
 * Same sizes and limits as jk_transition_pairwise_topk_forward (1 <= k <= 64, rp <= 128).
 * Replaces the scatter of low_rank_pairwise_topk_forward_cuda (jakal_net_native_cuda.cu:
 * 740-878, atomicAdd at :862-873) and of the blocked path jakal_net_native.cpp:6916-7087.
 */
int jk_transition_pairwise_topk_routes(const void* src_proj, const void* dst_proj, int64_t batch,
                                       int64_t n_src, int64_t n_dst, int64_t rp, int proj_dtype,
                                       const void* src_sender, int state_dtype, int64_t k,
                                       float score_bias, const float* bias_dev, int compress,
                                       float* routes, float* out_scores, int64_t* out_index,
                                       jk_stream_t stream);

/* Multi-head (jk_heads_t) variant of jk_transition_pairwise_topk_routes. */
int jk_transition_pairwise_topk_routes_mh(const void* src_proj, const void* dst_proj, int64_t batch,
                                          int64_t n_src, int64_t n_dst, int64_t rp, int proj_dtype,
                                          const void* src_sender, int state_dtype, int64_t k,
                                          float score_bias, const float* bias_dev, int compress,
                                          float* routes, float* out_scores, int64_t* out_index,
                                          const jk_heads_t* heads, jk_stream_t stream);

/*
 * Select-aggregate over materialised f32 score rows (any k, any score rank):
 *   scores [B, row_count, n_cols] holds score[b, t, s] for the rows t in
 *   [row_begin, row_begin + row_count) of an n_rows-row operator (e.g. a plain GEMM of the
 *   projections). Visibility, selection (ties to the lower column), score_bias / bias_dev,
 *   compressors and sender weighting are those of jk_propagation_topk_forward, with no limit
 *   on k or on the rank that produced the scores.
 *   scatter == 0 (gather): out_state [B, n_rows] / out_val [B, n_rows, dim] (out_dtype) get
 *     rows row_begin..; state / sender [B, n_cols], val [B, n_cols, dim] are per column.
 *   scatter == 1 (per-source transition): rows are sources; state / sender [B, n_rows],
 *     val [B, n_rows, dim]; acc_state [B, n_cols] and acc_val [B, n_cols, dim] (f32, zeroed
 *     by the caller) receive sum_t w[t, s] * state[t] and sum_t w[t, s] * val[t, :].
 *   sel_score f32 / sel_index int64 [B, row_count, k] (caller scratch, also a result): the
 *   selected scores (bias included) and columns in ascending column order, -inf / -1 pad.
 * One CTA per row: an exact 4-pass radix select over order-preserving keys, block prefix
 * sums for the survivors, block reductions for the compressor, then the gather or the
 * scatter. Replaces the blocked top-k paths that take any k:
 * jakal_net_native.cpp:6390-6447 (propagation_topk), :6916-7087 (transition_pairwise_topk)
 * and :7089-7246 (transition_query_topk), the path the reference takes when its CUDA kernels
 * refuse k > 64 (jakal_net_native_cuda.cu:2432-2434, 2557-2559).
 */
int jk_select_aggregate_forward(const float* scores, int64_t batch, int64_t n_rows, int64_t n_cols,
                                int64_t row_begin, int64_t row_count, const void* state,
                                const void* sender, int state_dtype, const void* val, int64_t dim,
                                int val_dtype, int64_t k, int64_t window, float score_bias,
                                const float* bias_dev, int compress, int scatter, void* out_state,
                                void* out_val, int out_dtype, float* acc_state, float* acc_val,
                                float* sel_score, int64_t* sel_index, jk_stream_t stream);

/* ---- backward (training) kernels --------------------------------------------------
 * The row-wise pieces of the top-k operators' backward, behind the reference's autograd
 * Functions (native_backend.py:4408-4601 uses softmax_backward_cuda and the reduce
 * backward; the kernels replaced are jakal_net_native_cuda.cu:2112-2320). `dtype` applies to
 * every tensor argument of a call (JK_F32, JK_BF16, JK_F16); accumulation is f32.
 */

/* grad_scores[r, j] = routes[r, j] * (grad_routes[r, j] - sum_j' routes[r, j'] grad_routes[r, j'])
 * for rows x n row-major tensors (the softmax backward; jakal_net_native.cpp:408-416). */
int jk_softmax_backward(const void* routes, const void* grad_routes, void* grad_scores, int64_t rows,
                        int64_t n, int dtype, jk_stream_t stream);

/* grad_scores[i] = grad_edges[i] / (1 + |scores[i]|)^2 over n elements (softsign backward;
 * jakal_net_native.cpp:398-406). */
int jk_softsign_backward(const void* scores, const void* grad_edges, void* grad_scores, int64_t n,
                         int dtype, jk_stream_t stream);

/* Gather half of the backward of a top-k reduce (out[b, q] = sum_e edges[b, q, e] *
 * x[b, indices[b, q, e]]; jakal_net_native.cpp:152-166):
 *   grad_edges[b, q, e] = grad_state[b, q] * state[b, idx] + grad_val[b, q, :] . val[b, idx, :]
 * indices int64 [B, n_rows, k] (-1: no edge, gradient 0), state [B, n_src], val
 * [B, n_src, dim], grad_state [B, n_rows], grad_val [B, n_rows, dim] in dtype; grad_edges
 * [B, n_rows, k] in out_dtype. The scatter half (the gradients of state and val) is a GEMM of
 * the dense edge matrix (jk_topk_to_dense). */
int jk_topk_reduce_backward_edges(const int64_t* indices, const void* state, const void* val,
                                  const void* grad_state, const void* grad_val, void* grad_edges,
                                  int64_t batch, int64_t n_rows, int64_t n_src, int64_t k, int64_t dim,
                                  int dtype, int out_dtype, jk_stream_t stream);

/* dense[r, indices[r, e]] += w[r, e] for rows x k selections (f32 w, int64 indices, -1 and
 * zero weights skipped); dense f32 [rows, n_cols] zeroed by the caller. A selection names
 * each column once; padded window index lists may repeat a placeholder column with weight 0,
 * which adds nothing. Turns the scatters of the backward into GEMMs with a fixed summation
 * order. */
int jk_topk_to_dense(const float* w, const int64_t* indices, float* dense, int64_t rows, int64_t k,
                     int64_t n_cols, jk_stream_t stream);

/* ---- training-step kernels --------------------------------------------------------
 * The row and parameter operators around the propagation / transition operators in a training
 * step: the apply step of a layer (sum = x + scale * delta, then a layer norm;
 * progressive_b_example.py:71-99, 282-294), the loss over the query head's vocabulary and the
 * clipping of the gradients. dtype codes JK_F32, JK_BF16, JK_F16; strides count elements from
 * one row to the next (rows are contiguous inside); any alignment of a whole element. All
 * arithmetic is f32 or wider; a result is rounded once, to its own type. Results do not depend
 * on the order in which blocks run.
 */

/* Layer norm of sum = x + delta_scale * delta (delta NULL: of x):
 *   mean = E[sum], rstd = 1 / sqrt(E[(sum - mean)^2] + eps), y = (sum - mean) * rstd * weight + bias
 * x [rows, dim], delta [rows, dim] in dtype, weight / bias [dim] in param_dtype (NULL: 1 / 0);
 * out: y and sum [rows, dim] contiguous in dtype (sum may be NULL; the statistics and y are of
 * the unrounded sum), mean / rstd f32 [rows] (both or neither NULL). */
int jk_layer_norm_forward(const void* x, int64_t x_stride, const void* delta, int64_t delta_stride,
                          float delta_scale, const void* weight, const void* bias, int param_dtype,
                          int64_t rows, int64_t dim, int dtype, float eps, void* y, void* sum,
                          float* mean, float* rstd, jk_stream_t stream);

/* f32 elements of the workspace that jk_layer_norm_backward needs for its parameter gradients. */
int64_t jk_layer_norm_backward_workspace(int64_t rows, int64_t dim);

/* Backward of jk_layer_norm_forward. With n = (sum - mean) * rstd and u = grad_y * weight:
 *   grad_x = rstd * (u - E[u] - n * E[u * n]) + grad_sum,  grad_delta = delta_scale * grad_x,
 *   grad_weight = sum over rows of grad_y * n,             grad_bias = sum over rows of grad_y.
 * grad_sum (NULL: 0) is the gradient that reaches sum from its other uses; grad_x, grad_delta
 * [rows, dim] contiguous in dtype (grad_delta may be NULL); grad_weight and grad_bias [dim] in
 * param_dtype (both or neither NULL), summed over fixed blocks of rows in a fixed order.
 * workspace: jk_layer_norm_backward_workspace(rows, dim) floats, 16-byte aligned (may be NULL
 * without parameter gradients). */
int jk_layer_norm_backward(const void* grad_y, int64_t grad_y_stride, const void* sum, int64_t sum_stride,
                           const float* mean, const float* rstd, const void* weight, int param_dtype,
                           const void* grad_sum, int64_t grad_sum_stride, float delta_scale, int64_t rows,
                           int64_t dim, int dtype, void* grad_x, void* grad_delta, void* grad_weight,
                           void* grad_bias, float* workspace, jk_stream_t stream);

/* reduction codes of the cross entropy */
#define JK_REDUCE_NONE 0
#define JK_REDUCE_MEAN 1 /* over the rows whose target is not ignore_index */
#define JK_REDUCE_SUM 2

/* Bytes of the workspace of jk_cross_entropy_forward and _backward. */
int64_t jk_cross_entropy_workspace(int64_t rows);

/* Softmax cross entropy of logits [rows, vocab] (dtype, vocab <= 2^30) against targets int64 [rows]:
 *   lse = log sum_j exp(z_j),  loss = lse - (1 - a) z_target - a E_j[z_j]   (a = label_smoothing)
 * A row whose target is ignore_index is not read and has loss, lse and gradient 0; a target
 * outside [0, vocab) gives its row a NaN loss and gradient (nothing is read there). Logits of
 * -inf have probability 0; a row of nothing else has a NaN loss and gradient and an lse of -inf.
 * out: losses f32 [rows] and lse f32 [rows] (each may be NULL), loss f32 scalar by `reduction`
 * (NULL with JK_REDUCE_NONE; the mean over no row is NaN, the sum 0), and, when grad is not NULL
 * (not with JK_REDUCE_NONE), grad [rows, vocab] in dtype, in the same pass over the logits:
 *   grad = grad_scale * d loss / d logits = grad_scale * w * (softmax(z) - (1 - a) onehot - a / vocab)
 * with w = 1 (sum) or 1 / number of rows that count (mean). grad may be the logits themselves.
 * workspace: jk_cross_entropy_workspace(rows) bytes, 8-byte aligned. */
int jk_cross_entropy_forward(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows,
                             int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                             int reduction, float grad_scale, float* losses, float* lse, float* loss,
                             void* grad, int64_t grad_stride, void* workspace, jk_stream_t stream);

/* Gradient of the cross entropy from the lse that the forward pass kept:
 *   grad = g * w * (exp(z - lse) - (1 - a) onehot - a / vocab)
 * grad_loss: device f32, [rows] with JK_REDUCE_NONE (g per row, w = 1), else one value; grad
 * [rows, vocab] in dtype (may be the logits); rows to ignore get zeros. workspace:
 * jk_cross_entropy_workspace(rows) bytes, 8-byte aligned. */
int jk_cross_entropy_backward(const float* grad_loss, const void* logits, int64_t logits_stride,
                              const int64_t* targets, const float* lse, int64_t rows, int64_t vocab, int dtype,
                              int64_t ignore_index, float label_smoothing, int reduction, void* grad,
                              int64_t grad_stride, void* workspace, jk_stream_t stream);

/* The same two with the log-sum kept in two f32, lse + lse_low (f32 [rows]; lse_low may be NULL, as 0):
 * a gradient from one f32 is off by a factor of exp(half a unit in its last place), which matters for
 * logits far from 0 (2^-11 at 1e4; at 1e8 neighbouring logits are not told apart). The forward form is
 * the loss alone. */
int jk_cross_entropy_forward_split(const void* logits, int64_t logits_stride, const int64_t* targets, int64_t rows,
                                   int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                   int reduction, float* losses, float* lse, float* lse_low, float* loss,
                                   void* workspace, jk_stream_t stream);
int jk_cross_entropy_backward_split(const float* grad_loss, const void* logits, int64_t logits_stride,
                                    const int64_t* targets, const float* lse, const float* lse_low, int64_t rows,
                                    int64_t vocab, int dtype, int64_t ignore_index, float label_smoothing,
                                    int reduction, void* grad, int64_t grad_stride, void* workspace,
                                    jk_stream_t stream);

/* norm codes of jk_clip_grad_norm */
#define JK_NORM_2 0
#define JK_NORM_INF 1

/* Bytes of the workspace of jk_clip_grad_norm. */
int64_t jk_clip_grad_norm_workspace(void);

/* Norm over all elements of `count` flat tensors, and their clipping:
 *   total = sqrt(sum g^2) (JK_NORM_2; squares are added in f32 by up to 32, in f64 where that would
 *           leave f32's range, and their sums in f64, so they neither overflow nor vanish) or
 *           max |g| (JK_NORM_INF), NaN if any element is;
 *   out_i = g_i * min(1, max_norm / (total + eps)).
 * grads, outs, numels, dtypes, out_dtypes are HOST arrays of `count` entries that are read
 * during the call; outs NULL: in place (then a coefficient of 1 writes nothing). clip 0: the norm
 * alone (outs, max_norm, eps unused). total: device f32 scalar. workspace:
 * jk_clip_grad_norm_workspace() bytes, 16-byte aligned. Tensors must not overlap. */
int jk_clip_grad_norm(const void* const* grads, void* const* outs, const int64_t* numels, const int* dtypes,
                      const int* out_dtypes, int64_t count, int norm_kind, int clip, float max_norm, float eps,
                      float* total, void* workspace, jk_stream_t stream);

/* ---- generation-step kernels ------------------------------------------------------
 * What a model that produces one node after another needs: the propagation of a few new nodes
 * over the nodes that a paged cache holds, the pages themselves, and the verification of drafted
 * tokens. No reference counterpart: the reference computes whole layers (its query-block model
 * drafts a block of tokens at once, progressive_b_example.py:2059-2152).
 *
 * A cache: pools [pages, ...] whose dim 0 is the page (keys [pages, kv_heads, page_size, rank],
 * values [.., dim], states [pages, kv_heads, page_size], one set per layer); table int32
 * [batch, columns]: the page of nodes [c * page_size, (c + 1) * page_size) of a sequence, -1: none;
 * lengths int32 [batch]; refs int32 [pages]: how many table entries name a page (0: it is free).
 * Table entries outside [0, pages) are as -1: nothing is read or written there. Calls on one cache
 * go on one stream, or are ordered by events. Strides count elements unless they say bytes.
 */

/* The cache of a call. refs may be NULL where it is not named below. */
typedef struct jk_cache {
  int32_t* table;
  int64_t table_stride;
  int32_t* lengths;
  int32_t* refs;
  int64_t batch, columns, pages, page_size;
} jk_cache_t;

/* Nodes to propagate: query [batch, new_nodes, heads, rank]; keys, values, states [pages, kv_heads,
 * page_size, rank | dim | -], last dim contiguous, strides of the dims before it (query: sequence, node,
 * head; else page, head, place) in elements; states NULL: none, then out_state is NULL. All in
 * dtype, any alignment of an element. out_value [batch, new_nodes, heads, dim] and out_state
 * [batch, new_nodes, heads] contiguous in dtype. workspace: jk_cached_propagation_workspace(...) bytes,
 * 16-byte aligned. */
typedef struct jk_nodes {
  const void* query;
  int64_t query_stride[3];
  const void* keys;
  int64_t key_stride[3];
  const void* values;
  int64_t value_stride[3];
  const void* states;
  int64_t state_stride[3];
  const int32_t* counts;
  int64_t new_nodes, heads, kv_heads, rank, dim, dtype, window, compress;
  void* out_value;
  void* out_state;
  void* workspace;
} jk_nodes_t;

/* Bytes of the workspace of jk_cached_propagation (0: none is needed). */
int64_t jk_cached_propagation_workspace(int64_t batch, int64_t new_nodes, int64_t heads, int64_t kv_heads,
                                        int64_t rank, int64_t dim, int64_t page_size, int64_t columns,
                                        int64_t window, int dtype);

/* Propagation of the last n = counts[b] (NULL: new_nodes; clamped to [0, new_nodes]) nodes of every
 * sequence over the nodes before them and themselves. Node t of the n is at place
 * p = lengths[b] - n + t and sees the places j <= p that are in the cache, j >= p - window
 * (window < 0: all); head h reads the cache's head h / (heads / kv_heads):
 *   s_j = scale * query[b, t, h] . keys[j] + score_bias,  w = compress(s) over the visible j
 *   out_value[b, t, h] = sum_j w_j values[j],  out_state[b, t, h] = sum_j w_j states[j]
 * with compress JK_SOFTMAX, JK_SOFTSIGN or JK_SIGNED_ABS_SOFTMAX. A node that sees none, and nodes
 * t >= n, have zeros; a softmax over scores that are all -inf is NaN. What places that are not
 * seen hold (NaN, infinities) has no part in a result; a NaN score or an infinite value that is seen has the
 * part that the formula gives it. Sums are f32, before they are divided by the
 * weights' sum. 16-bit weights go into the value product as two planes, rounded by at most 2^-16 of a
 * weight, in f16 at least 2^-32 of the largest (softsign: 2^-40).
 * rank <= 256, dim <= 512, new_nodes <= 64, heads a multiple of kv_heads. */
int jk_cached_propagation(const jk_cache_t* cache, const jk_nodes_t* nodes, float scale, float score_bias,
                          jk_stream_t stream);

/* Pools of a call: HOST arrays of `count` entries (at most 512), read during the call: the pools'
 * addresses, the bytes of a page and the bytes from one page to the next. */
typedef struct jk_pools {
  void* const* data;
  const int64_t* page_bytes;
  const int64_t* stride_bytes;
  int64_t count;
} jk_pools_t;

/* Bytes of the workspace of jk_cache_reserve. */
int64_t jk_cache_reserve_workspace(int64_t batch, int64_t pages);

/* Room for counts[b] more nodes in every sequence, in the order of the sequences: pages that are
 * free when the call begins, lowest first, enter the table with one reference; lengths grow. A
 * sequence that grows inside a page that others hold too (refs > 1) first gets a copy of that page
 * in every pool and gives up its reference. added[b] (int32 [batch]) is counts[b], or 0 where the
 * sequence is left as it is: a negative count, more nodes than the table's row has room for or than
 * 2^31 - 65, or pages that ran out (from the first sequence that could not be served on, none that needs a page
 * is). Needs refs. workspace: jk_cache_reserve_workspace(...) bytes, 16-byte aligned. */
int jk_cache_reserve(const jk_pools_t* pools, const jk_cache_t* cache, const int32_t* counts, int32_t* added,
                     void* workspace, jk_stream_t stream);

/* Rows to write, rows[i] [batch, new_nodes, heads, width] into pages[i] [pages, heads, page_size, width]
 * for `count` (at most 64) pairs. HOST arrays: addresses; strides, three a tensor (page, head, place;
 * sequence, node, head) in elements; widths; element sizes in bytes (1, 2, 4, 8). Rows are contiguous
 * inside. */
typedef struct jk_rows {
  void* const* pages_data;
  const int64_t* pages_strides;
  const void* const* rows_data;
  const int64_t* rows_strides;
  const int64_t* widths;
  const int64_t* element_bytes;
  int64_t count, new_nodes, heads;
} jk_rows_t;

/* Node t < n = counts[b] (NULL: new_nodes; clamped to [0, new_nodes]) of sequence b goes to place
 * lengths[b] - n + t, if the table has a page for it. */
int jk_cache_write(const jk_rows_t* rows, const jk_cache_t* cache, const int32_t* counts, jk_stream_t stream);

/* Bytes of the workspace of jk_cache_fork. */
int64_t jk_cache_fork_workspace(int64_t batch, int64_t forks);

/* Sequence children[i] becomes a copy of sequence parents[i] as that was when the call began; its
 * pages are shared (one more reference each). done[i] (bytes, 0 or 1) is 0, and nothing happens,
 * where a number is outside the batch, the child is not empty (length 0), or an earlier i names the
 * same child. Needs refs. workspace: jk_cache_fork_workspace(...) bytes, 16-byte aligned. */
int jk_cache_fork(const jk_cache_t* cache, const int32_t* parents, const int32_t* children, int64_t forks,
                  uint8_t* done, void* workspace, jk_stream_t stream);

/* Sequences are cut to new_lengths[b] nodes (clamped to [0, lengths[b]]): table entries past the last
 * page that is still needed give up their references and become -1. new_lengths may be lengths.
 * Needs refs. */
int jk_cache_release(const jk_cache_t* cache, const int32_t* new_lengths, jk_stream_t stream);

/* Bytes of the workspace of jk_cache_compact. */
int64_t jk_cache_compact_workspace(int64_t pages);

/* Moves the pages in use (refs > 0) to the front: with live of them, the i-th in use at or past `live`
 * goes to the i-th free one before it, in every pool; table and refs follow, live (device int32)
 * receives their number. The pages that were moved from keep their contents. Needs refs (lengths may
 * be NULL). workspace: jk_cache_compact_workspace(pages) bytes, 16-byte aligned. */
int jk_cache_compact(const jk_pools_t* pools, const jk_cache_t* cache, int32_t* live, void* workspace,
                     jk_stream_t stream);

/* pool[dst[i]] = pool[src[i]] in every pool, for int32 src, dst [n]; pairs with a number outside
 * [0, pages) are left out. A page may be read by several pairs; one that a pair writes may be neither
 * read nor written by another pair of the call (its contents are then not defined). */
int jk_cache_copy(const jk_pools_t* pools, const int32_t* src, const int32_t* dst, int64_t n, int64_t pages,
                  jk_stream_t stream);

/* Drafted tokens: target [batch, drafted + 1, vocab] and draft [batch, drafted, vocab] (NULL: the draft is
 * certain of its tokens) in dtype, rows contiguous, strides of the first two dims in elements; tokens
 * int64 [batch, drafted], uniform f32 [batch, drafted + 1], contiguous; counts int32 [batch] or NULL.
 * out_tokens int64 [batch, drafted + 1], accepted int32 [batch]. */
typedef struct jk_draft {
  const void* target;
  int64_t target_stride[2];
  const void* draft;
  int64_t draft_stride[2];
  const int64_t* tokens;
  const float* uniform;
  const int32_t* counts;
  int64_t batch, drafted, vocab, dtype;
  int64_t* out_tokens;
  int32_t* accepted;
} jk_draft_t;

/* Verification of drafted tokens. Sequence b has n = counts[b] (NULL: drafted; clamped to [0, drafted])
 * drafted tokens x_i, drawn from draft[b, i, :], and the target's probabilities target[b, i, :] for
 * i <= n. Token i is accepted while uniform[b, i] * draft[b, i, x_i] < target[b, i, x_i] (exact; draft
 * NULL: probability 1); with the first a that is not (a = n: all are), out_tokens[b, a] is the least j with
 *   sum_{j' <= j} r_j' > uniform[b, drafted] * sum r,
 * r = max(target[b, a] - draft[b, a], 0) for a < n (target[b, a] where that is 0 throughout), target[b, n]
 * for a = n, in f64. NaN and negative values count as 0 (infinite ones leave the new token open); a token outside the vocabulary is not
 * accepted; where r has no positive entry out_tokens[b, a] is -1. Before it stand the accepted tokens,
 * behind it -1; accepted[b] is a. vocab <= 2^30. */
int jk_verify_draft(const jk_draft_t* draft, jk_stream_t stream);

/* Failure-path test entry (no reference counterpart): jk_propagation_window_forward
 * (softsign, no bias) with a producer warp that issues no load and no MMA, so every consumer
 * wait runs into its bound (about 2 s): the kernel sets the device error word, releases its
 * TMEM and returns; jk_device_status then reports JK_ERR_DEVICE_TIMEOUT and the context stays
 * usable. Outputs are zeros. For tests of that path only. */
int jk_debug_window_stalled_producer(const void* row_proj, const void* col_proj, int64_t batch,
                                     int64_t n_rows, int64_t n_cols, int64_t rp, int proj_dtype,
                                     const void* col_state, int state_dtype, const void* col_val,
                                     int64_t dim, int64_t window, void* out_state, void* out_val,
                                     int out_dtype, jk_stream_t stream);

/*
 * Allocation-free per-source sparse transition. No counterpart in the reference: it exists
 * for callers that cannot allocate device memory at call time -- plain-C / FFI hosts with no
 * device allocator of their own, and latency-critical loops that must not call cudaMalloc /
 * cudaFree because those can synchronise the device. Same contract as
 * jk_transition_pairwise_topk_forward without the `accum` argument: the f32 scratch is a
 * fixed 16 MiB device array inside the library (held on every GPU that loads it until exit),
 * so B * n_dst * (dim + 1) must not exceed jk_transition_pairwise_topk_noalloc_capacity()
 * floats, else JK_ERR_BAD_SHAPE. Every call looks up the array's address on the current
 * device (so it stays valid after a device reset or from another context); the first call
 * on a device also loads the library's module there, so make it before any stream capture. Calls share the array: calls that overlap on the GPU
 * race; serialise them on one stream. The scratch is zeroed on the stream by every call.
 */
int jk_transition_pairwise_topk_forward_noalloc(const void* src_proj, const void* dst_proj,
                                                int64_t batch, int64_t n_src, int64_t n_dst,
                                                int64_t rp, int proj_dtype, const void* src_state,
                                                const void* src_sender, int state_dtype,
                                                const void* src_val, int64_t dim, int val_dtype,
                                                int64_t k, float score_bias, const float* bias_dev,
                                                int compress, void* out_state, void* out_val,
                                                int out_dtype, jk_stream_t stream);

/* Scratch capacity (in f32 elements) of the allocation-free entry point above. */
int64_t jk_transition_pairwise_topk_noalloc_capacity(void);

#ifdef __cplusplus
}
#endif

#endif /* JAKAL_B200_H_ */
