/*
 * rmoe.h - C ABI of the MI355X-native quantized sparse-MoE block.
 *
 * All tensor pointers are caller-owned DEVICE pointers (for instance the
 * data_ptr() of torch tensors on the GPU); every compute call is enqueued on
 * `stream` (a hipStream_t passed as void*, NULL = the default stream) and
 * returns without waiting for the GPU.  Every call returns RMOE_OK (0) or a
 * negative RMOE_E* code; the message for the last failure on the calling
 * thread is rmoe_last_error().  Arguments are validated on the host before
 * anything is launched, so argument errors never reach the GPU.  No call
 * allocates device memory: scratch space is the caller's `workspace`,
 * which must be zero-filled once when it is first allocated (the library
 * keeps its counters at a fixed offset and leaves them at zero when each
 * call completes, so one workspace serves calls of any shape) and must not
 * be shared by calls that may run concurrently.
 *
 * Weight format (MLX "affine", transpose=True): a matrix W[out, in] of
 * `bits`-bit codes is stored as uint32 words [out, in * bits / 32], element
 * k of a row in word k / (32/bits) at bit offset bits * (k % (32/bits)),
 * least-significant first; scales and biases are bf16 [out, in / group];
 * W[r, k] = q * scale + bias.  Expert banks add a leading [experts] axis.
 * bf16 values travel as uint16_t bit patterns.
 *
 * Reference interfaces replaced (paths relative to the waylake/runnel tree):
 *   rmoe_switch_glu   FusedQuantizedSwitchGLU.__call__   src/runnel/mlx.py:57-82
 *   rmoe_gather_qmm   mx.gather_qmm / QuantizedSwitchLinear, called at
 *                     src/runnel/mlx.py:64-75 and :77-79
 *   rmoe_moe_block    mlx-lm SparseMoeBlock.__call__ (the caller of the
 *                     module, invoked as layer.mlp(x) at
 *                     bench/mlx_component_profile.py:130)
 *   rmoe_router       the router half of that block (gate -> softmax ->
 *                     top-k -> renormalise)
 *   rmoe_router_q     the same with the 8-bit QuantizedLinear gate of real
 *                     checkpoints (bench/runnel_bench/checkpoint.py:200-208)
 *   rmoe_quantize / rmoe_dequantize
 *                     mx.quantize / mx.dequantize (affine, group 64), the
 *                     format produced for the banks that
 *                     src/runnel/mlx.py:38-48 concatenates
 *   rmoe_stream_read  the HBM stream calibrator that replaces
 *                     native/shaders/persistent_stream.metal:12-79
 */
#ifndef RMOE_H
#define RMOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RMOE_ABI_VERSION 7

#define RMOE_OK 0
#define RMOE_EINVAL (-1) /* inconsistent or unsupported shape / argument */
#define RMOE_EBITS (-2)  /* bits not in {4, 8} or group size not 64 */
#define RMOE_EALIGN (-3) /* a pointer is not 16-byte aligned */
#define RMOE_EWS (-4)    /* workspace missing or too small */
#define RMOE_EHIP (-5)   /* the HIP runtime reported an error */
#define RMOE_ENULL (-6)  /* a required pointer is NULL */
/* Not returned by any call (the calls do not wait for the GPU): the codes
 * callers report when a workspace's status word (rmoe_workspace_status_offset)
 * is 1 (a single-launch decode gave up a cross-workgroup wait, or the call
 * was cancelled) or 2 (a workgroup read an XCC id outside 0-7, so it could
 * not take part in the XCD-local hand-overs). */
#define RMOE_ETIMEOUT (-7)
#define RMOE_EPLACEMENT (-8)

/* One MLX-affine quantized bank: w [experts, rows, cols*bits/32] u32,
 * scales / biases [experts, rows, cols/group_size] bf16. */
typedef struct rmoe_qweight {
  const uint32_t* w;
  const uint16_t* scales;
  const uint16_t* biases;
  int32_t experts;
  int32_t rows;
  int32_t cols;
  int32_t bits;
  int32_t group_size;
} rmoe_qweight;

/* One MoE layer's resident weights.  gate_up rows are [up; gate]
 * (src/runnel/mlx.py:38-48).  The shared expert is present when
 * shared_gate_up.w != NULL; shared_gate_w (bf16 [hidden]) is its sigmoid
 * gate.  norm_topk_prob != 0 renormalises the selected probabilities.
 *
 * The router gate is either bf16 (router_w) or an 8-bit group-64 MLX-affine
 * bank (router_q, [1, experts, hidden]; router_w NULL), the format real
 * checkpoints give mlp.gate and mlp.shared_expert_gate
 * (bench/runnel_bench/checkpoint.py:200-208,
 * bench/results/m0/checkpoint-ornith-mlx-8bit.json:163-175).  The shared
 * gate then uses the same format: shared_gate_q [1, 1, hidden] instead of
 * shared_gate_w.  Quantized gate logits follow a fixed fp32 order of their
 * own: 16-code chunks lane + 64 i of a 64-lane wave, per chunk
 * acc = fma(sum q x, s, acc), acc = fma(sum x, b, acc), then a butterfly.
 *
 * post_norm_w != NULL puts the decoder layer's post-attention RMSNorm in
 * front of the block (appended in ABI version 3): the block's input is
 * rmoe_rms_norm(x, post_norm_w, norm_eps), the residual stays what the
 * caller passes, so a decoder computes h' = h + MoE(RMSNorm(h)) with
 * residual = x = h (the layer sequence of docs/architecture.md:31-37).
 *
 * Shapes: hidden and inter multiples of 64; hidden at most 4096 at 8 bits
 * (8192 at 4 bits); inter / (16 at 8 bits, 32 at 4 bits) a power of two
 * <= 64; experts <= 1024; top_k <= min(64, experts). */
typedef struct rmoe_layer {
  int32_t hidden;
  int32_t inter;
  int32_t shared_inter;
  int32_t experts;
  int32_t top_k;
  int32_t norm_topk_prob;
  const uint16_t* router_w;      /* bf16 [experts, hidden] */
  const uint16_t* shared_gate_w; /* bf16 [hidden], or NULL */
  rmoe_qweight gate_up;          /* [experts, 2*inter, hidden] */
  rmoe_qweight down;             /* [experts, hidden, inter] */
  rmoe_qweight shared_gate_up;   /* [1, 2*shared_inter, hidden] */
  rmoe_qweight shared_down;      /* [1, hidden, shared_inter] */
  rmoe_qweight router_q;         /* 8-bit gate [1, experts, hidden], or w NULL */
  rmoe_qweight shared_gate_q;    /* 8-bit shared gate [1, 1, hidden], or w NULL */
  const uint16_t* post_norm_w;   /* bf16 [hidden] RMSNorm weights, or NULL */
  float norm_eps;                /* its epsilon, in [0, 1] */
} rmoe_layer;

int rmoe_abi_version(void);

/* RMSNorm of `tokens` rows (mx.fast.rms_norm(x, weight, eps); checkpoints
 * store the effective weight): out = bf16(bf16(x r) w) with r = 1 /
 * sqrt(sum(x^2) / hidden + eps), the sum in the router's fixed fp32 order,
 * r correctly rounded.  hidden a multiple of 8; x, weight, out bf16, 16-byte
 * aligned. */
int rmoe_rms_norm(const uint16_t* x, const uint16_t* weight, int32_t tokens, int32_t hidden,
                  float eps, uint16_t* out, void* stream);

/* (This call and rmoe_swiglu came with ABI version 6.)
 * out[t] = bf16(sum_j weights[t, j] y[t, j] + sigmoid(gate[t]) shared[t]) in
 * fp32, the slots in order, then the shared expert's row; with a residual
 * bf16(residual[t] + that).  The tail of mlx-lm's block around a SwitchGLU
 * (bench/mlx_lm_adapter.py:49-94) for rows that are already computed.
 * y bf16 [tokens, top_k, hidden], weights fp32 [tokens, top_k], shared bf16
 * [tokens, hidden] with its gate's logits bf16 [tokens], or both NULL;
 * hidden a multiple of 8; row arrays 16-byte aligned. */
int rmoe_combine(const uint16_t* y, const float* weights, int32_t tokens, int32_t top_k,
                 int32_t hidden, const uint16_t* shared, const uint16_t* gate,
                 const uint16_t* residual, uint16_t* out, void* stream);

/* out = bf16(bf16(silu(gate)) * up) over n bf16 values (mlx-lm SwiGLU on
 * separate projections); 16-byte aligned. */
int rmoe_swiglu(const uint16_t* up, const uint16_t* gate, int64_t n, uint16_t* out,
                void* stream);

const char* rmoe_last_error(void);
const char* rmoe_status_string(int status);

/* Host-only validation of a layer description (no GPU access). */
int rmoe_validate_layer(const rmoe_layer* layer);

/* Bytes of workspace the block / router / switch calls need for `tokens`. */
size_t rmoe_workspace_bytes(const rmoe_layer* layer, int32_t tokens);

/* Router of mlx-lm's SparseMoeBlock: bf16 logits x . router_w^T (fixed fp32
 * reduction order), top_k experts by (logit desc, index asc), softmax over
 * all experts, probabilities rounded to bf16, renormalised when
 * norm_topk_prob.  indices int32 [tokens, top_k] in rank order, scores
 * fp32 [tokens, top_k] (bf16-valued). */
int rmoe_router(const uint16_t* router_w, int32_t experts, int32_t hidden,
                int32_t top_k, int32_t norm_topk_prob, const uint16_t* x,
                int32_t tokens, int32_t* indices, float* scores,
                void* workspace, size_t workspace_bytes, void* stream);
size_t rmoe_router_workspace_bytes(int32_t experts, int32_t top_k,
                                   int32_t tokens);

/* The same router with an 8-bit group-64 quantized gate (mlx-lm's
 * QuantizedLinear gate, x @ dequantize(W)^T): router [1, experts, hidden]
 * (experts = router->rows, hidden = router->cols), logits in the quantized
 * gate's fixed fp32 order.  Workspace: rmoe_router_workspace_bytes. */
int rmoe_router_q(const rmoe_qweight* router, int32_t top_k, int32_t norm_topk_prob,
                  const uint16_t* x, int32_t tokens, int32_t* indices, float* scores,
                  void* workspace, size_t workspace_bytes, void* stream);

/* FusedQuantizedSwitchGLU.__call__ (src/runnel/mlx.py:57-82): for every
 * (token, slot) the packed [up; gate] projection of expert indices[t, j],
 * SwiGLU, then the expert's down projection.  y bf16 [tokens, top_k,
 * hidden], per slot and not combined.  A slot whose index is outside
 * [0, experts) yields a zero row and touches no weight memory.  From 64
 * (token, slot) rows on (the expert-sorted path) y must be 16-byte
 * aligned. */
int rmoe_switch_glu(const rmoe_qweight* gate_up, const rmoe_qweight* down,
                    const uint16_t* x, int32_t tokens, const int32_t* indices,
                    int32_t top_k, uint16_t* y, void* workspace,
                    size_t workspace_bytes, void* stream);
size_t rmoe_switch_workspace_bytes(const rmoe_qweight* gate_up,
                                   const rmoe_qweight* down, int32_t tokens,
                                   int32_t top_k);

/* The routed half of the block for a caller's routing: the experts of
 * rmoe_switch_glu, then out[t] = bf16(sum_j weights[t, j] * y[t, j]) in slot
 * order, with residual != NULL out[t] = bf16(residual[t] + out[t]).  mlx-lm's
 * `(switch_mlp(x, inds) * scores[..., None]).sum(-2)` (the caller of
 * src/runnel/mlx.py:57-82), and the reference's native two-stage MoE with
 * given router weights (native/src/fused_moe_probe.mm:494-537, the
 * RNLMOE01 datasets of bench/export_ornith_moe_layer.py).  weights fp32
 * [tokens, top_k]; a slot with an out-of-range index adds nothing; out bf16
 * [tokens, hidden], not aliasing x. */
int rmoe_switch_combine(const rmoe_qweight* gate_up, const rmoe_qweight* down,
                        const uint16_t* x, int32_t tokens, const int32_t* indices,
                        const float* weights, int32_t top_k, const uint16_t* residual,
                        uint16_t* out, void* workspace, size_t workspace_bytes,
                        void* stream);
size_t rmoe_switch_combine_workspace_bytes(const rmoe_qweight* gate_up,
                                           const rmoe_qweight* down, int32_t tokens,
                                           int32_t top_k);

/* gather_qmm(x, w, scales, biases, rhs_indices, transpose=True):
 * y[m] = x[lhs[m]] . deq(w[rhs[m]])^T for m < rows.  lhs_indices == NULL
 * means row m reads x[m]; rhs_indices == NULL means expert 0; a row whose
 * index is out of range is written as zeros.  x bf16 [x_rows, w->cols];
 * exactly one of y_bf16 / y_f32 ([rows, w->rows]) is non-NULL.  Each row
 * is a group-affine dot over fp32 weights fl32(q*s + b), except a dense
 * product (no index arrays) of 64 or more rows into a 16-byte aligned
 * y_bf16 with w->rows a multiple of 256 and w->cols a multiple of 128
 * (mx.quantized_matmul at prefill sizes, the reference's qmm_4d_tile,
 * native/shaders/quantized_qmm.metal:68-151): that one runs on the matrix
 * cores with every dequantised weight rounded to bf16 and fp32
 * accumulation.  Calls of many rows share an expert's weights between rows;
 * their fp32 sums run in another order than those of few, so a row's last
 * bits may differ between calls of different row counts.  Within a call a
 * row's value depends on that row alone, and equal calls give equal bits. */
int rmoe_gather_qmm(const uint16_t* x, int32_t x_rows,
                    const int32_t* lhs_indices, const int32_t* rhs_indices,
                    int32_t rows, const rmoe_qweight* w, uint16_t* y_bf16,
                    float* y_f32, void* stream);

/* Whole block (mlx-lm SparseMoeBlock.__call__): out[t] = bf16(sum_j
 * score_j * y_j + bf16(sigmoid(x . shared_gate_w)) * y_shared); with
 * residual != NULL, out[t] = bf16(residual[t] + out[t]).  indices_out /
 * scores_out may be NULL.  x, residual, out bf16 [tokens, hidden]; out may
 * alias residual but not x.  One token of a layer with hidden 2048, inter
 * 512, top_k <= 8 and experts <= 256 runs as one single-launch kernel on a
 * device of at least 256 CUs in 8 XCDs, such as MI355X (see
 * rmoe_workspace_status_offset); other calls that route fewer than 64
 * (token, slot) rows take the router, gate/up and down kernels; calls that
 * route 64 or more take the expert-sorted path, which needs out and
 * residual 16-byte aligned (2 bytes otherwise). */
int rmoe_moe_block(const rmoe_layer* layer, const uint16_t* x, int32_t tokens,
                   const uint16_t* residual, uint16_t* out,
                   int32_t* indices_out, float* scores_out, void* workspace,
                   size_t workspace_bytes, void* stream);

/* rmoe_moe_block without a workspace, for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference (its
 * probes own every buffer).  The call allocates nothing: its scratch is a
 * static device array of RMOE_NOALLOC_SCRATCH_BYTES held by each GPU the
 * library runs on until the process ends; a call that needs more
 * (rmoe_workspace_bytes(layer, tokens) > RMOE_NOALLOC_SCRATCH_BYTES, e.g.
 * long prefills) is refused with RMOE_EWS before anything is launched.
 * Every call on one GPU shares that array: calls that may overlap on one
 * GPU (different streams, different host threads) race and must be
 * serialised by the caller.  Arguments and outputs as rmoe_moe_block;
 * status_out (device uint32, may be NULL) receives this call's status word
 * (nonzero: a single-launch decode gave up a cross-workgroup wait and the
 * outputs are not valid), which the call then clears. */
#define RMOE_NOALLOC_SCRATCH_BYTES ((size_t)16 << 20)
int rmoe_moe_block_noalloc(const rmoe_layer* layer, const uint16_t* x, int32_t tokens,
                           const uint16_t* residual, uint16_t* out,
                           int32_t* indices_out, float* scores_out, uint32_t* status_out,
                           void* stream);

/* Batch-1 decode of one token through a stack of MoE layers with a residual
 * add between them: x_{l+1} = bf16(x_l + block_l(x_l)), one launch for the
 * whole stack (the chained decode of the reference's 40-layer model,
 * docs/architecture.md:31-37; there is no single reference entry point).
 * The layer descriptors are packed once on the host with
 * rmoe_chain_table_pack into rmoe_chain_table_bytes(n) bytes, copied by the
 * caller to device memory, and passed as device_table; layer0 describes the
 * common shape.  Needs hidden 2048, inter 512, top_k <= 8 (plus an optional
 * shared expert), experts <= 256 and a device of at least 256 CUs in 8 XCDs
 * (RMOE_EINVAL otherwise); rmoe_chain_table_pack checks the shape without
 * touching the device.  x, out bf16 [hidden]. */
size_t rmoe_chain_table_bytes(int32_t n_layers);
int rmoe_chain_table_pack(const rmoe_layer* layers, int32_t n_layers,
                          void* host_table);
int rmoe_moe_chain(const rmoe_layer* layer0, const void* device_table,
                   int32_t n_layers, const uint16_t* x, uint16_t* out,
                   void* workspace, size_t workspace_bytes, void* stream);

/* Byte offset inside a workspace of a uint32 status word: nonzero when a
 * single-launch decode or a few-token call (2-8 tokens at the single-launch
 * shapes, whose router hands its logits over between workgroups) failed
 * (the call still completes; its outputs are then not valid): 1 when a
 * workgroup gave up a cross-workgroup wait (every wait is bounded, and the
 * other workgroups of the call stop waiting as soon as one gives up), 2 when
 * a workgroup read an XCC id outside 0-7.  The word is sticky: later calls
 * leave it set until the caller clears it.  The uint32 before it holds the
 * workspace's phase epoch and the one after it the abort word: a caller
 * cancels the next such call on the workspace before it runs by writing
 * epoch + 1 there (the call then waits for nothing and sets the status word
 * to 1). */
size_t rmoe_workspace_status_offset(void);

/* Launch mode of the single-launch decode kernel (rmoe_moe_block with one
 * token of the decode shape, rmoe_moe_chain) outside stream capture.
 * enabled = 0 (the default): a plain launch, as stream capture records it
 * (a one-token layer call takes about 14 us back to back on MI355X);
 * workgroups that wait for others that are not yet resident (kernels of
 * other streams holding CUs) wait until those run, and two single-launch
 * calls that overlap on different streams can each hold CUs the other
 * needs: their waits then give up and set the status word above.
 * enabled = 1: a cooperative launch, which guarantees every workgroup is
 * resident whatever else runs on the device, but does not overlap the
 * previous call (about 18 us more per call), for callers that run such
 * calls on several streams at once.  Process-wide; returns the previous
 * mode.  No counterpart in the reference (its probes submit one Metal
 * command buffer per call). */
int rmoe_set_cooperative_launch(int32_t enabled);

/* Affine quantization of fp32 rows [rows, cols] (group_size 64, bits 4|8):
 * per group, the larger-magnitude edge value is kept exact, scale and bias
 * are rounded to bf16 and the codes are round-half-even((w - b) / s)
 * clipped to [0, 2^bits - 1]. */
int rmoe_quantize(const float* w, int64_t rows, int32_t cols, int32_t bits,
                  int32_t group_size, uint32_t* wq, uint16_t* scales,
                  uint16_t* biases, void* stream);

/* Dequantize rows [row_begin, row_begin + rows) of the flattened bank
 * (experts * rows) to fp32 fl32(q*s + b) (out_f32) and/or to bf16 of that
 * value (out_bf16); either output may be NULL. */
int rmoe_dequantize(const rmoe_qweight* w, int64_t row_begin, int64_t rows,
                    float* out_f32, uint16_t* out_bf16, void* stream);

/* Reads `bytes` (a multiple of 16) once with 16-byte loads using `blocks`
 * workgroups of 256 lanes; workgroup i folds what it read into partials[i]
 * (device uint32 [blocks], overwritten).  Measures achievable HBM read
 * bandwidth for a given launch shape. */
int rmoe_stream_read(const void* buffer, size_t bytes, uint32_t* partials,
                     int32_t blocks, void* stream);

/* ---- The decoder layer's other half: the token mixer (came with ABI
 * version 7).  No counterpart in the reference, whose attention and linear
 * attention are mlx-lm's; the layers are those of docs/architecture.md:31-37.
 * The calls below keep no counters: their workspaces need no zero-fill and
 * hold nothing between calls.  A call's outputs and its workspace lie apart
 * from its inputs and from each other, except where an input is said to be
 * written in place. */

/* Rows of heads: value d of head h of row t is x[t * row_stride + h *
 * head_stride + d], bf16; x 16-byte aligned, strides multiples of 8. */
typedef struct rmoe_rows {
  const uint16_t* x;
  int64_t row_stride;
  int64_t head_stride;
  int32_t heads;
} rmoe_rows;

/* A paged key-value cache: value d of token i of page p and key head h is at
 * p * page_stride + h * head_stride + i * row_stride + d of k and of v
 * (values; 16-byte aligned bases, strides multiples of 16 bytes).  bits 16:
 * bf16; bits 8: e4m3 (fn), a value being k_scale (v_scale) times its code.
 * page_size a power of two, 8..1024; dim 64, 96, 128, 192 or 256. */
typedef struct rmoe_paged_cache {
  void* k;
  void* v;
  int64_t page_stride;
  int64_t head_stride;
  int64_t row_stride;
  int32_t pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t dim;
  int32_t bits;
  float k_scale; /* read at bits 8 */
  float v_scale;
} rmoe_paged_cache;

/* Which values of a head turn, and by which positions: the first 2 * half,
 * pair i by position[axis(i)] * inv_freq[i] (inv_freq device fp32 [half]).
 * Pair i is values (i, i + half), or (2 i, 2 i + 1) when `adjacent`.  axes
 * 1..4 with sections[0..axes) summing to half: the pairs' axes one section
 * after the other, or, when `woven`, axis i mod axes as long as that axis's
 * section has pairs left (i / axes < section) and axis 0 beyond; a woven
 * section of another axis may not exceed its turns.  half a multiple of 8,
 * at most 128. */
typedef struct rmoe_rotary_spec {
  const float* inv_freq;
  int32_t half;
  int32_t axes;
  int32_t sections[4];
  int32_t woven;
  int32_t adjacent;
} rmoe_rotary_spec;

/* One step's bookkeeping from lengths on the device.  cached / added int32
 * [requests] (negative counts as 0; at most 4096 requests): tokens that
 * request r holds, and tokens it takes in this step.  Its pages from entry
 * ceil(cached / page_size) of block_table row r on, as many as cached +
 * added tokens need and table_width has room for, come from free_pages
 * [free_count] in order of request, then entry; past the end of that list
 * the entry becomes -1.  Other entries are left as they were.
 * Written: cu_seqlens [requests + 1], the running sum of added; lengths
 * [requests] = cached + added; counts [3]: tokens, pages taken, pages that
 * were missing (sums that pass INT32_MAX stay there); and for each of `rows`
 * rows, the tokens of all requests one after the other: slots (page *
 * page_size + place in it, or -1 where the token has no page), positions
 * (cached + place among the request's new tokens) and request_of; rows
 * behind the last token get -1, 0 and -1. */
int rmoe_paged_tables(const int32_t* cached, const int32_t* added, int32_t requests,
                      int32_t* block_table, int64_t table_stride, int32_t table_width,
                      const int32_t* free_pages, int32_t free_count, int32_t page_size,
                      int32_t rows, int64_t* slots, int32_t* positions, int32_t* request_of,
                      int32_t* cu_seqlens, int32_t* lengths, int32_t* counts, void* stream);

/* Rotary positions: q_out [rows, q heads, dim] and k_out [rows, k heads, dim]
 * = the turned rows (angles in 64 bits, products fp32, one rounding), values
 * past 2 * half copied.  positions int32, axis a's at positions + a *
 * axis_stride.  dim a multiple of 8, at most 1024. */
int rmoe_rotary(const rmoe_rotary_spec* spec, const int32_t* positions, int64_t axis_stride,
                int32_t rows, int32_t dim, const rmoe_rows* q, uint16_t* q_out,
                const rmoe_rows* k, uint16_t* k_out, void* stream);

/* The same with the turned keys and the values v written into the cache:
 * row t at slot slots[t] (int64, as rmoe_paged_tables gives them); a row whose
 * slot is outside the cache's writes nothing there.  bits 8: e4m3 of x * fp32(1
 * / scale), to nearest even, saturating.  Rows with one slot in common leave
 * either's values. */
int rmoe_rotary_append(const rmoe_rotary_spec* spec, const int32_t* positions,
                       int64_t axis_stride, int32_t rows, const rmoe_rows* q, uint16_t* q_out,
                       const rmoe_rows* k, const rmoe_rows* v, const rmoe_paged_cache* cache,
                       const int64_t* slots, void* stream);

/* Attention of one new token of each request over its cached keys:
 * out [requests, q->heads, dim] = softmax_j(scale q.k_j) v_j over j <
 * lengths[r], with window > 0 over the last `window` of them; query heads
 * [h G, (h + 1) G) read key head h, G = q->heads / kv_heads.  block_table
 * int32 [requests, table_width] (row stride table_stride); lengths past
 * table_width * page_size end there.  Keys of a page outside [0, pages) do
 * not count, whatever the cache holds.  A request without keys gets zeros and
 * lse -inf.  lse fp32 [requests, q->heads] (natural logarithm of the sum of
 * exp(scale q.k)) may be NULL.  The probabilities are rounded to bf16 for
 * their product with v; all else is fp32.  workspace: at least
 * rmoe_paged_attention_workspace_bytes, 16-byte aligned. */
int rmoe_paged_attention(const rmoe_rows* q, const rmoe_paged_cache* cache,
                         const int32_t* block_table, int64_t table_stride, int32_t table_width,
                         const int32_t* lengths, int32_t requests, int32_t window, float scale,
                         uint16_t* out, float* lse, void* workspace, size_t workspace_bytes,
                         void* stream);
size_t rmoe_paged_attention_workspace_bytes(const rmoe_paged_cache* cache, int32_t q_heads,
                                            int32_t requests, int32_t table_width,
                                            int32_t window);

/* Linear attention with a decay for each head over packed sequences: rows
 * [cu_seqlens[r], cu_seqlens[r + 1]) are sequence r's, whose state S
 * [v heads, dk, dv] is state[i], i = state_index[r] (r itself when NULL):
 *   S <- exp(log_decay) S + k u^T,  out = scale S^T q  (after the token)
 *   u = v, or with beta  u = beta (v - (exp(log_decay) S)^T k)
 * value heads [h G, (h + 1) G) use q and k head h.  The final state goes to
 * state_out[i], which may be state.  i outside [0, slots): from zeros, and
 * not kept.  The indices of one call differ.  log_decay, beta fp32, value
 * (t, h) at t * row_stride + h * head_stride (0 repeats one); beta NULL: no
 * delta rule.  out bf16 [tokens, v heads, dv]; rows of no sequence become
 * zero with clear_uncovered and stay as they were without.  dk 64 or 128, dv
 * a multiple of 16, v heads a multiple of k's.  States stay fp32 throughout.
 * A NaN or infinity among a sequence's inputs may reach all of that
 * sequence's outputs, earlier tokens' too, and no other sequence's.
 * workspace: rmoe_linear_attention_workspace_bytes (0: the call needs none),
 * 16-byte aligned. */
typedef struct rmoe_gate {
  const float* x;
  int64_t row_stride;
  int64_t head_stride;
} rmoe_gate;
int rmoe_linear_attention(const rmoe_rows* q, const rmoe_rows* k, const rmoe_rows* v,
                          const rmoe_gate* log_decay, const rmoe_gate* beta,
                          const int32_t* cu_seqlens, int32_t tokens, int32_t requests,
                          int32_t dk, int32_t dv, float scale, const float* state,
                          float* state_out, const int32_t* state_index, int32_t slots,
                          uint16_t* out, int32_t clear_uncovered, void* workspace,
                          size_t workspace_bytes, void* stream);
size_t rmoe_linear_attention_workspace_bytes(int32_t tokens, int32_t requests, int32_t k_heads,
                                             int32_t v_heads, int32_t dk, int32_t delta);

#ifdef __cplusplus
}
#endif

#endif /* RMOE_H */
