/*
 * libmusapy_b200 - musapy's stride-aware elementwise and reduction engine
 * for NVIDIA B200 (sm_100a). Public C-ABI.
 *
 * Two families of entry points:
 *
 *  1. Extended entry points (mpb_*): one call per musapy operator, a dtype tag
 *     per operand (promotion casts are fused into the kernels), an int status
 *     return, caller-owned scratch. These are what the Python surface
 *     (musapy_b200) binds, and what a host layer in any language should bind.
 *     They replace the per-dtype kernel wrappers that musapy's operator layer
 *     calls from rust/musapy-ops/src/op_builder.rs (launch_binary! ...
 *     launch_argreduce_partial!, :38-223, and the cast/cumsum dispatch at
 *     :968-1045 and :3321-3330).
 *
 *  2. Reference-named kernel symbols (musapy_<op>_<dtype>_v2 / _v3), declared
 *     in include/musapy_kernels_v2.h: the exact set and signatures of
 *     rust/musapy-ops/src/kernels.rs:16-343, so a CUDA build of musapy's Rust
 *     layers can link this library unchanged.
 *
 * Conventions (shared with musapy's kernel contract, docs/adr/ADR.md:322-338):
 *  - strides and offsets are in ELEMENTS and may be 0 (broadcast) or negative
 *    (flipped views); each data pointer addresses the logical element
 *    [0, ..., 0] of its view (the view offset is already applied);
 *  - outputs are C-contiguous;
 *  - shape / stride arrays are host memory read during the call only;
 *  - every launch is asynchronous on `stream`; the library never allocates
 *    device memory (scratch is passed in) and never synchronises, except
 *    mpb_cumsum_status which reads a status word back;
 *  - dtype tags follow musapy's Dtype enum order
 *    (rust/musapy-core/src/dtype.rs:25-41), see enum mpb_dtype.
 */
#ifndef MUSAPY_B200_H
#define MUSAPY_B200_H

#include <stddef.h>
#include <stdint.h>

#include "mpb_types.h"

#ifdef __cplusplus
extern "C" {
#endif

/* cudaStream_t without requiring the CUDA headers. */
typedef struct CUstream_st* mpb_stream_t;

/* ---------------------------------------------------------------- status */

/* Message describing the last non-OK status returned on this thread. */
const char* mpb_last_error(void);
/* ABI version of this header (bumped on incompatible changes). */
int mpb_version(void);
/* Multiprocessor count of the current device (148 on B200; 148 without a device). */
int mpb_num_sms(void);
/* Number of kernels this library has launched in the process so far. */
unsigned long long mpb_launch_count(void);

/* ------------------------------------------------------- host-side helpers */

/* Result dtype of a binary op: rust/musapy-core/src/dtype.rs:302-338
 * (`promote`); all_gpu=1 selects the narrow-first rule musapy applies when
 * every input lives on the device. Returns -1 when no promotion exists. */
int mpb_promote(int a_dtype, int b_dtype, int all_gpu);

/* NumPy broadcast of two shapes: rust/musapy-ops/src/broadcast.rs:24-58
 * (`broadcast_shape`). Writes max(na, nb) extents to `out`; returns that
 * ndim, or -1 when the shapes are incompatible. */
int mpb_broadcast_shape(int na, const int64_t* a_shape, int nb, const int64_t* b_shape, int64_t* out);

/* Strides of an operand against a broadcast target:
 * rust/musapy-ops/src/broadcast.rs:71-92 (`broadcast_strides`). */
void mpb_broadcast_strides(int ndim, const int64_t* shape, const int64_t* strides, int target_ndim,
                           const int64_t* target, int64_t* out);

/* The engine's dimension collapsing (replaces the per-element offset_nd of
 * kernels/include/common.h:42-51): drops extent-1 dims and merges adjacent
 * dims that every operand allows. `strides` holds nops x ndim values;
 * writes the collapsed shape and nops x result strides; returns the
 * collapsed ndim (>= 1), or -1 on bad arguments. Host only. */
int mpb_collapse(int ndim, const int64_t* shape, int nops, const int64_t* strides, int64_t* out_shape,
                 int64_t* out_strides);

/* Kernel class the reduction planner picks (1 row_warp, 2 row_block,
 * 3 row_split, 4 col, 5 col_split, 6 gen; 0 empty) and the output count M,
 * reduced length L and split count. Host only; negative status on error. */
int mpb_reduce_plan(int ndim, const int64_t* shape, const int64_t* strides, int in_dtype, uint64_t axes_mask,
                    int64_t* M, int64_t* L, int64_t* splits);

/* mpb_reduce_plan for reduction `op` (an mpb_red_op) of an input at address
 * `a` (the column kernels' vector width depends on the op and on the
 * address's alignment), also giving the outputs each thread of a column
 * kernel (kinds 4 and 5) reduces: 1, or 2/4/8 when every group of them is
 * one aligned 8- or 16-byte load at every reduced step. No counterpart in
 * the reference (its column kernels take one output per thread). Host only;
 * `a` is not dereferenced. */
int mpb_reduce_plan_at(int op, int ndim, const int64_t* shape, const int64_t* strides, const void* a, int in_dtype,
                       uint64_t axes_mask, int64_t* M, int64_t* L, int64_t* splits, int* outputs_per_thread);

/* ------------------------------------------------------------ elementwise */

/* out = op(a[, b]) over `shape`, for every mpb_ew_op:
 *   MPB_ADD..MPB_POW   binary arithmetic; replaces musapy_{add,sub,mul,div,pow}
 *                      _{f32,f64,c64,c128}_v2 (rust/musapy-ops/src/kernels.rs:19-28,
 *                      :102-109) plus the cast temporaries of op_builder.rs:410-417
 *   MPB_EQ..MPB_GE     comparisons, out_dtype MPB_BOOL (kernels.rs:84-95, :114-117)
 *   MPB_SIN..MPB_NEG   unary math (kernels.rs:31-44, :110-113)
 *   MPB_CLAMP          p0 = lo, p1 = hi (kernels.rs:47-48)
 *   MPB_CAST           dtype conversion / strided copy (kernels.rs:51-81, :119-124)
 *   MPB_FILL           out = p0 (+ i*p1 for complex); a and b unused
 * a_strides / b_strides are already broadcast to `shape` (0 on broadcast
 * dims); b is NULL for unary ops. compute_dtype is the promoted dtype the op
 * is evaluated in; a and b are read in their own dtypes and converted in
 * registers. */
int mpb_elementwise(int op, int ndim, const int64_t* shape, const void* a, int a_dtype, const int64_t* a_strides,
                    const void* b, int b_dtype, const int64_t* b_strides, void* out, int out_dtype,
                    int compute_dtype, double p0, double p1, mpb_stream_t stream);

/* Transposed-view elementwise ops (an input with unit stride on an outer
 * dim) run through TMA tile loads when the view's layout allows it (16-byte
 * aligned base and strides, 2-, 4- or 8-byte elements); mpb_ew_set_tma(0)
 * routes them to the shared-memory tile kernel instead, (1) back, (-1)
 * queries. Returns the previous setting. No counterpart in musapy. */
int mpb_ew_set_tma(int enable);

/* TMA-tiled kernel launches in this process so far. */
uint64_t mpb_ew_tma_launches(void);

/* Synchronous: *timed_out = 1 when a TMA tile wait gave up (2 s) since the
 * last call on this device (the op's output is then incomplete), else 0;
 * clears the flag. No counterpart in musapy. */
int mpb_ew_wait_status(int* timed_out);

/* -------------------------------------------------------------- reductions */

/* Device scratch (bytes) mpb_reduce needs for this request; 0 when none. */
size_t mpb_reduce_scratch_bytes(int op, int ndim, const int64_t* shape, const int64_t* strides, const void* a,
                                int in_dtype, uint64_t axes_mask, int compute_dtype);

/* Reduce the dims set in axes_mask (bit d = dim d) with an mpb_red_op.
 * Replaces the naive / small_axis / partial / mid / final kernel families of
 * kernels.rs:139-180, :222-304 and the host path choice of
 * op_builder.rs:2310-3139 with one call. The output is C-contiguous over the
 * kept dims in order. nan_first_rule=1 applies musapy's CPU rule for
 * max/min/argmax/argmin (a NaN is the answer only when it is the first
 * element). Multiple axes reduce in one pass; argmax/argmin over several axes
 * report the flat index over those axes (reduction.rs:186-223). Integer
 * inputs narrower than 64 bits must be widened to int64 by the caller (as
 * musapy's cast_array does); MPB_R_ARGMAX_REC / _ARGMIN_REC write a 16-byte
 * {value bits, index} record per output for cross-shard combining. */
int mpb_reduce(int op, int ndim, const int64_t* shape, const int64_t* strides, const void* a, int in_dtype,
               uint64_t axes_mask, void* out, int out_dtype, int compute_dtype, int nan_first_rule, void* scratch,
               size_t scratch_bytes, mpb_stream_t stream);

/* Same as mpb_reduce but with no scratch argument: the scratch comes from an
 * array built into the library (256 KiB per GPU, held from the library's
 * load on that GPU until the process exits). No counterpart in musapy. It
 * exists for callers that cannot allocate device memory: an application that
 * embeds this library and owns the whole device budget through its own pool,
 * or a latency-critical loop in which cudaMalloc / cudaFree must not run
 * because they can synchronise the device. It allocates nothing. No request
 * is refused for its size: the reduction splits across CTAs only as far as
 * its partials fit in the 256 KiB (a reduction with more than 16384 outputs
 * runs unsplit, which needs no scratch). Where that limit changes the split,
 * float sums and means may differ from mpb_reduce's in the last bits;
 * otherwise both run the same plan and agree bit for bit. All calls on a GPU
 * share the array and it keeps the last call's contents (nothing in it needs
 * to start at zero), so calls that can overlap on the GPU race: order them on
 * one stream or with events. The first call on each device looks up the
 * array's device address with that device current; make that first call
 * before any stream capture begins (later uncaptured calls look it up again,
 * so a device reset is picked up). */
int mpb_reduce_noalloc(int op, int ndim, const int64_t* shape, const int64_t* strides, const void* a, int in_dtype,
                       uint64_t axes_mask, void* out, int out_dtype, int compute_dtype, int nan_first_rule,
                       mpb_stream_t stream);

/* ------------------------------------------------------------------ cumsum */

/* Device scratch (bytes) mpb_cumsum needs; 0 when none. */
size_t mpb_cumsum_scratch_bytes(int ndim, const int64_t* shape, const int64_t* strides, const void* a, int in_dtype,
                                int axis, void* out, int out_dtype);

/* Inclusive prefix sum along `axis`; out_dtype is the compute dtype (f32,
 * f64, or i64 for integer inputs). Replaces musapy_cumsum_{i64,f32,f64}_v3
 * (kernels.rs:185-187) without its 256^3 length limit. The scratch is
 * cleared by the call itself. */
int mpb_cumsum(int ndim, const int64_t* shape, const int64_t* strides, const void* a, int in_dtype, int axis,
               void* out, int out_dtype, void* scratch, size_t scratch_bytes, mpb_stream_t stream);

/* Synchronises `stream` and reads the status word a look-back cumsum left in
 * its scratch: MPB_OK, or MPB_ERR_TIMEOUT when a bounded wait gave up. */
int mpb_cumsum_status(const void* scratch, mpb_stream_t stream);

/* ------------------------------------------- recurrent block operators */

/* The operators below are new: musapy has no counterpart. Element types are
 * MPB_F32, MPB_F16 and MPB_BF16, arithmetic is in float, outputs are
 * C-contiguous, the innermost stride of every input is 1 and the other
 * strides are given in elements. Scratch is 16-byte aligned; what a call
 * leaves in it is of no use to the next. */

/* Gated linear recurrence over time. x is (B, T, D) with strides x_sb, x_st
 * over sequences and steps; gate is (B, T, H), H a divisor of D (channel d
 * has gate d / (D / H)), of x's type or MPB_F32; h0 (B, D) floats or NULL for
 * zero. mode MPB_SCAN_LINEAR: h[t] = g h[t-1] + x[t]; MPB_SCAN_SIGMOID:
 * h[t] = s h[t-1] + (1 - s) x[t], s = sigmoid(g). Linear gates may exceed one;
 * what shrinks below 2^-126 of itself within 128 steps may be lost. Writes h (B, T, D) in x's
 * type and, when state is not NULL, h[T-1] (h0 when T == 0) in float; state
 * may not overlap h0. Scratch: mpb_gated_scan_scratch_bytes(..., backward = 0). */
size_t mpb_gated_scan_scratch_bytes(int64_t B, int64_t T, int64_t D, int64_t H, int x_dtype, int gate_dtype,
                                    int backward);
int mpb_gated_scan(int64_t B, int64_t T, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, int64_t x_st,
                   const void* gate, int gate_dtype, int64_t g_sb, int64_t g_st, const float* h0, int mode, void* h,
                   float* state, void* scratch, size_t scratch_bytes, mpb_stream_t stream);

/* Gradients of mpb_gated_scan from dh (B, T, D), the gradient of every h[t],
 * and dstate (B, D) or NULL, that of the last state in float. h is the
 * forward pass's output as it stored it, h0 what it started from. Writes dx
 * (B, T, D), dgate (B, T, H, summed over a gate's channels in a fixed order,
 * in the gate's type; zeros when D == 0) and dh0 (B, D) in float when not NULL. */
int mpb_gated_scan_backward(int64_t B, int64_t T, int64_t D, int64_t H, const void* dh, int64_t dh_sb, int64_t dh_st,
                            const void* x, int x_dtype, int64_t x_sb, int64_t x_st, const void* gate, int gate_dtype,
                            int64_t g_sb, int64_t g_st, const void* h, int64_t h_sb, int64_t h_st, const float* h0,
                            const float* dstate, int mode, void* dx, void* dgate, float* dh0, void* scratch,
                            size_t scratch_bytes, mpb_stream_t stream);

/* Synchronises `stream` and reads the status word that a scan left in its
 * scratch (NULL: it had none): MPB_OK, or MPB_ERR_TIMEOUT when a bounded wait between
 * the pieces of a long sequence gave up (the results from there on are NaN). */
int mpb_gated_scan_status(const void* scratch, mpb_stream_t stream);

/* One step of B running sequences: x (B, D), gate (B, H); updates state
 * (B, D) in place and writes the new state in x's type to h (B, D). */
int mpb_gated_scan_step(int64_t B, int64_t D, int64_t H, const void* x, int x_dtype, int64_t x_sb, const void* gate,
                        int gate_dtype, int64_t g_sb, int mode, float* state, void* h, mpb_stream_t stream);

/* Norms before and after a block with its gate, dropout and residual scale,
 * over R rows of D, less than 2^29 elements apart: n = z rms(z) w_post; y = x + scale * drop(act(gate) n);
 * u = y rms(y) w_pre, rms(v) = (mean v^2 + eps)^(-1/2). x, z, gate in
 * `dtype` with row strides x_sr, z_sr, g_sr; gate_kind says the gate's extent
 * (mpb_gate_kind), activation what it goes through (mpb_activation); the
 * weights are D floats. dropout > 0 drops elements of the branch as
 * mpb_dropout does, by their index in (R, D). Writes y and u (R, D) and
 * rstd (2, R): the two rms factors, NaN when D == 0. z == NULL: the plain norm
 * u = x rms(x) w_pre, no y, rstd (1, R). */
int mpb_gated_residual_norm(int64_t R, int64_t D, int dtype, const void* x, int64_t x_sr, const void* z, int64_t z_sr,
                            const void* gate, int64_t g_sr, int gate_kind, int activation, const float* w_post,
                            const float* w_pre, double scale, double eps, double dropout, uint64_t seed,
                            uint64_t offset, void* y, void* u, float* rstd, mpb_stream_t stream);

/* Gradients of mpb_gated_residual_norm from dy and du (each may be NULL for
 * zero), with y and rstd as the forward pass left them and the same gate,
 * scale, dropout, seed and offset. Writes dx, dz (R, D), dgate (the gate's
 * extent, its type) and the weights' gradients (D floats), summed in a fixed
 * order. z == NULL: the plain norm's gradients (y is its input; dz, dgate and
 * dw_post unused). */
size_t mpb_gated_residual_norm_scratch_bytes(int64_t R, int64_t D, int dtype, int branch, int gate_kind);
int mpb_gated_residual_norm_backward(int64_t R, int64_t D, int dtype, const void* dy, int64_t dy_sr, const void* du,
                                     int64_t du_sr, const void* y, int64_t y_sr, const void* z, int64_t z_sr,
                                     const void* gate, int64_t g_sr, int gate_kind, int activation,
                                     const float* w_post, const float* w_pre, const float* rstd, double scale,
                                     double dropout, uint64_t seed, uint64_t offset, void* dx, void* dz, void* dgate,
                                     float* dw_post, float* dw_pre, void* scratch, size_t scratch_bytes,
                                     mpb_stream_t stream);

/* Dropout of n contiguous elements: element i is dropped when its 16 bits of
 * a Philox-4x32-10 stream (counter {i / 8, offset}, key seed, half i % 8) are
 * below k = floor(p * 65536 + 1/2), else multiplied by 65536 / (65536 - k).
 * The gradient is the same call on the output's gradient. */
int mpb_dropout(int64_t n, const void* x, int dtype, double p, uint64_t seed, uint64_t offset, void* y,
                mpb_stream_t stream);

/* Clipped policy loss with a KL term over N tokens of V logits (row stride
 * l_sr) and, when dlogits is not NULL, its gradient times grad_scale. targets
 * are N MPB_I32 or MPB_I64 indices; old_logp, advantages, ref_logp (NULL: no
 * KL term) N floats; mask N bytes or NULL. Writes the mean loss over the mask,
 * logp, kl (N floats), clipped (N bytes) and dlogits (N, V) in `dtype`;
 * tokens outside the mask give zeros whatever their logits and target hold;
 * a target outside [0, V) gives NaN. */
size_t mpb_policy_loss_scratch_bytes(int64_t N, int64_t V, int dtype);
int mpb_policy_loss(int64_t N, int64_t V, const void* logits, int dtype, int64_t l_sr, const void* targets,
                    int targets_dtype, const float* old_logp, const float* advantages, const float* ref_logp,
                    const void* mask, double clip_low, double clip_high, double kl_coef, double grad_scale, float* loss,
                    float* logp, float* kl, void* clipped, void* dlogits, void* scratch, size_t scratch_bytes,
                    mpb_stream_t stream);

/* ------------------------------------- recurrent language model operators */

/* New too, with the conventions of the operators above. */

/* Linear attention with a decay for each head. q and k are (B, T, Hq, DK) and v
 * is (B, T, H, DV), Hq a divisor of H (head h has q and k of head h / (H / Hq)), in
 * `dtype` with strides over sequences, steps and heads; log_decay is (B, T, H)
 * floats with strides g_sb, g_st, g_sh (0 repeats it). From state0 (B, H, DK, DV)
 * floats, NULL for zero:
 *   S = e^log_decay S + k v',   o = scale S' q.
 * Writes o (B, T, H, DV) and, when state is not NULL, the last S (state0 when T == 0); state may
 * not overlap state0. A log-decay below -104 is a decay of zero: what came before has no part from there on.
 * Channels per head: 1 to 256. Scratch: mpb_linear_attention_scratch_bytes; it is less where `aligned` says that q, k, v and o
 * (backward: q, k, v and dout) are 16-byte aligned with strides that are positive multiples of 16 bytes, and has to be asked
 * for so or not as the call's are. Backward it holds the state and its gradient at every 64th step, T DK DV / 8 bytes per
 * sequence and head; forward, but for aligned MPB_BF16 heads of up to 128 channels, the state. Values are finite: one that
 * is not may reach every result of its chunk of 64 steps and the later ones. What decays leave below 2^-102 keeps fewer
 * bits, and below 2^-126 none. */
size_t mpb_linear_attention_scratch_bytes(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype,
                                          int backward, int decay_by_head, int aligned);
int mpb_linear_attention(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* q,
                         int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                         const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const float* log_decay, int64_t g_sb,
                         int64_t g_st, int64_t g_sh, const float* state0, double scale, void* o, float* state, void* scratch,
                         size_t scratch_bytes, mpb_stream_t stream);

/* Synchronises `stream` and reads the status word that a call left in its scratch (NULL: it had none): MPB_OK, or
 * MPB_ERR_TIMEOUT when a bounded wait between the warps of a block gave up (its results, and what is made
 * from its states, are NaN). */
int mpb_linear_attention_status(const void* scratch, mpb_stream_t stream);

/* How long such a wait may take, in nanoseconds (in steps of 4000), in the calls from now on, of every thread: two seconds
 * at most, and unless this says otherwise; 0 lets every wait give up at once, to test what follows. Returns the limit before. */
int64_t mpb_linear_attention_wait_limit(int64_t ns);

/* Gradients of mpb_linear_attention from dout (B, T, H, DV) and dstate (B, H, DK, DV) floats or NULL, that of the
 * last state. Writes dq and dk (B, T, Hq, DK, summed over the heads that share one), dv (B, T, H, DV), dlog_decay
 * (B, T, H) floats, or with decay_by_head (H) floats, summed over sequences and steps in a fixed order, and
 * dstate0 (B, H, DK, DV) floats, which may not overlap dstate. */
int mpb_linear_attention_backward(int64_t B, int64_t T, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* dout,
                                  int64_t do_sb, int64_t do_st, int64_t do_sh, const void* q, int64_t q_sb, int64_t q_st,
                                  int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st, int64_t k_sh, const void* v,
                                  int64_t v_sb, int64_t v_st, int64_t v_sh, const float* log_decay, int64_t g_sb, int64_t g_st,
                                  int64_t g_sh, const float* state0, const float* dstate, double scale, void* dq, void* dk,
                                  void* dv, float* dlog_decay, int decay_by_head, float* dstate0, void* scratch,
                                  size_t scratch_bytes, mpb_stream_t stream);

/* One step of B running sequences: q and k (B, Hq, DK), v (B, H, DV), log_decay (B, H); updates state (B, H, DK, DV)
 * floats, 16-byte aligned, in place and writes o (B, H, DV). */
int mpb_linear_attention_step(int64_t B, int64_t H, int64_t Hq, int64_t DK, int64_t DV, int dtype, const void* q, int64_t q_sb,
                              int64_t q_sh, const void* k, int64_t k_sb, int64_t k_sh, const void* v, int64_t v_sb, int64_t v_sh,
                              const float* log_decay, int64_t g_sb, int64_t g_sh, double scale, float* state, void* o,
                              mpb_stream_t stream);

/* Distillation from a teacher's top logits: N tokens of V logits (row stride l_sr) in `dtype`; ids (N, K) MPB_I32 or
 * MPB_I64 places in the vocabulary and teacher (N, K) the teacher's logits there (MPB_F32, MPB_F16 or MPB_BF16),
 * C-contiguous, K at most 1024. Per token kl = sum p (log p - log q), p the softmax of the K over the temperature
 * (0.001 to 1000), q that of the V; loss = temperature^2 times the mean over the mask (N bytes or NULL). Writes kl
 * (N floats), the loss and, when dlogits is not NULL, the gradient of grad_scale * loss (N, V) in `dtype`. Entries of
 * -inf are left out whatever their id; a token without entries gives zeros, a place outside [0, V) or a NaN
 * entry NaN, tokens outside the mask zeros whatever they hold. */
size_t mpb_distill_loss_scratch_bytes(int64_t N);
int mpb_distill_loss(int64_t N, int64_t V, int64_t K, const void* logits, int dtype, int64_t l_sr, const void* ids,
                     int ids_dtype, const void* teacher, int teacher_dtype, const void* mask, double temperature,
                     double grad_scale, float* loss, float* kl, void* dlogits, void* scratch, size_t scratch_bytes,
                     mpb_stream_t stream);

/* Rows of a table (V, D) in `dtype`, row stride t_sr, for N tokens (MPB_I32 or MPB_I64), times a scale, to out (N, D);
 * a token outside [0, V) gives a row of NaN. */
int mpb_embedding(int64_t N, int64_t V, int64_t D, const void* table, int dtype, int64_t t_sr, const void* tokens,
                  int tokens_dtype, double scale, void* out, mpb_stream_t stream);

/* The table's gradient from dout (N, D) in `dtype`, row stride d_sr: scale times the sum, in their order, of the rows
 * whose token names a row, in float. Writes dtable (V, D) floats whole, or with `into` adds to it where tokens name a
 * row. Tokens outside [0, V) have no part. */
size_t mpb_embedding_backward_scratch_bytes(int64_t N, int64_t V, int64_t D, int into);
int mpb_embedding_backward(int64_t N, int64_t V, int64_t D, const void* dout, int dtype, int64_t d_sr, const void* tokens,
                           int tokens_dtype, double scale, int into, float* dtable, void* scratch, size_t scratch_bytes,
                           mpb_stream_t stream);

/* ---------------------------------------------------------------- creation */

/* Fills `out` (n contiguous elements of `dtype`) with start + i*step, each
 * value evaluated in f64 (multiply, then add, each rounded) and converted once
 * with Rust `as` semantics, as the CPU path of ms.arange does
 * (creation.rs:469-501 and :324-348). Replaces musapy_arange_{f32,f64,i64,i32}
 * (kernels.rs, init.mu:86-97), which compute in the element type; every dtype
 * is accepted. The caller derives n from start/stop/step (arange_len,
 * creation.rs:624-633). */
int mpb_arange(void* out, int dtype, int64_t n, double start, double step, mpb_stream_t stream);

/* n evenly spaced values from start to stop inclusive: step = (stop - start) /
 * (n - 1) in f64, element i = start + i*step as in mpb_arange; n == 1 gives
 * start (creation.rs:508-521 and :350-377). Replaces musapy_linspace_{f32,f64}
 * (init.mu:102-115). */
int mpb_linspace(void* out, int dtype, int64_t n, double start, double stop, mpb_stream_t stream);

/* rows x cols matrix (C-contiguous) of zeros with ones where col - row == k
 * (creation.rs:457-461, init.mu:47-56). Replaces musapy_eye_{f32,f64,i64,i32}
 * (init.mu:121-134); every dtype is accepted. */
int mpb_eye(void* out, int dtype, int64_t rows, int64_t cols, int64_t k, mpb_stream_t stream);

/* --------------------------------------------------- host <-> device copies */

/* Copies `bytes` from pageable (or any) host memory to device memory `dst`
 * on `stream`, through a ring of pinned staging slots with the host-side
 * copies spread over a few threads and overlapped with the DMA of the
 * previous chunk; a page-locked source (cudaHostAlloc / cudaHostRegister) is
 * moved by one DMA with no staging. Returns once the host source has been read completely (it
 * may be reused at once); the device copy completes in stream order. Replaces
 * the list-based host transfer of ms.array (rust/musapy-python/src/ops.rs:
 * 354-625) and the plain musaMemcpy behind it (musa_ffi.rs). The device is the
 * current CUDA device. */
int mpb_copy_h2d(void* dst, const void* src, size_t bytes, mpb_stream_t stream);

/* Copies `bytes` of device memory `src` to host memory `dst` after the work
 * already queued on `stream`, and returns when `dst` holds the data. Same
 * staging ring as mpb_copy_h2d, the DMA of chunk k+4 overlapping the host
 * copy of chunk k; a page-locked destination gets one DMA, no staging. Replaces Array.tolist's transfer (array.rs:451-488). */
int mpb_copy_d2h(void* dst, const void* src, size_t bytes, mpb_stream_t stream);

/* ---------------------------------------------------- axis-0 sharding (new) */

/* Device combine of per-rank argmax/argmin records (MPB_R_ARG*_REC output,
 * all-gathered in rank order) into one global flat index; rank_offsets[r] is
 * the flat index of rank r's first element. No counterpart in musapy, which
 * has no multi-GPU path. */
int mpb_shard_arg_combine(const int64_t* records, int nranks, const int64_t* rank_offsets, int is_max, int is_int,
                          int64_t* out_index, double* out_value, mpb_stream_t stream);

/* Writes sum and mean (true global count) of an all-reduced f64 total in the
 * array dtype (MPB_F32 or MPB_F64). No counterpart in musapy. */
int mpb_shard_sum_finalize(const double* total, double count, int out_dtype, void* sum_out, void* mean_out,
                           mpb_stream_t stream);

/* ------------------------------------------- peer record exchange (new) */

/* Record exchange over NVLink peer memory between the ranks of one node, the
 * last step of a sharded full reduction. No counterpart in musapy, which has
 * no multi-GPU path. Each rank allocates one exchange buffer
 * (mpb_peer_alloc: cudaMalloc of mpb_peer_buffer_bytes() bytes, zeroed, plus
 * its CUDA IPC handle of mpb_peer_handle_bytes() bytes), the handles are
 * exchanged out of band, and each rank opens the others (mpb_peer_open). */
size_t mpb_peer_buffer_bytes(void);
size_t mpb_peer_handle_bytes(void);
int mpb_peer_alloc(void** buf, void* ipc_handle);
int mpb_peer_open(const void* ipc_handle, void** peer_buf);
int mpb_peer_close(void* peer_buf);
int mpb_peer_free(void* buf);

/* Exchange number `seq` (1, 2, ... the same sequence on every rank): stores
 * this rank's `rec_bytes` (8, 16, 24 or 32) record into every rank's buffer
 * (peers[r] is rank r's buffer as mapped here, peers[rank] the local one),
 * then waits until all `world` records of this exchange have arrived and
 * writes them to `out` in rank order (world x rec_bytes, 8-byte aligned).
 * Records travel as flag-in-line words (each 8-byte half of a 16-byte
 * store is {4 data bytes, 32-bit seq}), so no fence or flag store is
 * needed. Waits are bounded (~2 s): on expiry *status (device int) becomes
 * MPB_ERR_TIMEOUT and the kernel returns without writing `out`. At most 16
 * ranks. */
int mpb_peer_allgather(const void* rec, int rec_bytes, void* const* peers, int rank, int world, uint64_t seq,
                       void* out, int* status, mpb_stream_t stream);

/* The exchange of mpb_peer_allgather fused with the finish of a sharded
 * sum: `partial` is this rank's f64 partial sum; the `world` partials are
 * summed in rank order (the same value on every rank) and the sum and mean
 * (over `count` elements) written in MPB_F32 or MPB_F64. One kernel. No
 * counterpart in musapy. */
int mpb_peer_sum_finalize(const double* partial, void* const* peers, int rank, int world, uint64_t seq, double count,
                          int out_dtype, void* sum_out, void* mean_out, int* status, mpb_stream_t stream);

/* The exchange fused with the finish of a sharded argmax / argmin: `record`
 * is this rank's {value bits, local index} (MPB_R_ARG*_REC output); the
 * records are combined in rank order as mpb_shard_arg_combine does
 * (rank_offsets[r] = flat index of rank r's first element). One kernel. No
 * counterpart in musapy. */
int mpb_peer_arg_combine(const int64_t* record, void* const* peers, int rank, int world, uint64_t seq,
                         const int64_t* rank_offsets, int is_max, int is_int, int64_t* out_index, double* out_value,
                         int* status, mpb_stream_t stream);

/* The two fused exchanges above with all `world` ranks played on ONE GPU:
 * one cooperative launch of `world` blocks (every block resident at once),
 * block r acting as rank r with exchange buffer bufs[r] (zeroed
 * mpb_peer_buffer_bytes() buffers on this GPU), record partials[r] /
 * records[2r..2r+1] and results sum_out[r], mean_out[r] (f32 or f64 per
 * out_dtype) / out_index[r], out_value[r]. The kernels, wire format, waits
 * and combine are those of the per-rank calls; only the launch differs.
 * For checking the multi-rank exchange and combine where fewer GPUs than
 * ranks exist (ranks that wait on one another must never be separate
 * launches on one GPU). No counterpart in musapy. */
int mpb_peer_sum_finalize_emulated(const double* partials, void* const* bufs, int world, uint64_t seq, double count,
                                   int out_dtype, void* sum_out, void* mean_out, int* status, mpb_stream_t stream);
int mpb_peer_arg_combine_emulated(const int64_t* records, void* const* bufs, int world, uint64_t seq,
                                  const int64_t* rank_offsets, int is_max, int is_int, int64_t* out_index,
                                  double* out_value, int* status, mpb_stream_t stream);

/* Sum of `world` f64 partials (stride_bytes apart) in rank order, then sum
 * and mean (over `count` elements) in MPB_F32 or MPB_F64. No counterpart in
 * musapy. */
int mpb_shard_sum_parts_finalize(const double* parts, int stride_bytes, int world, double count, int out_dtype,
                                 void* sum_out, void* mean_out, mpb_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MUSAPY_B200_H */
