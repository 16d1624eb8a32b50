/*
 * adhip -- C ABI of the MI355X (gfx950) execution backend for the autodiff-ir-rust `Device` interface.
 *
 * Every entry point is what a Rust `HipDevice` (an `impl Device`, reference src/core/ir.rs:126-143) binds
 * over FFI.  Plain pointers and sizes only; no exceptions or panics cross this boundary: functions return
 * 0 on success and a non-zero code on failure, with the message available from adhip_last_error().
 *
 * A context is used by one thread at a time (the reference holds its DEVICE mutex around every call,
 * src/core/ir.rs:180-198, src/core/value.rs:83-91).
 */
#ifndef ADHIP_H
#define ADHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct adhip_ctx adhip_ctx;
typedef struct adhip_program adhip_program;

/* Library version string. */
const char* adhip_version(void);

/* Open HIP device `device_ordinal` and create a context (one stream).
 * Replaces OpenCL::new(CLDeviceType) -- reference src/devices/opencl/device.rs:41-58. */
int adhip_create(int device_ordinal, adhip_ctx** out);

/* Release the context, its compiled kernels, the programs it kept and its result buffers. */
void adhip_destroy(adhip_ctx* ctx);

/* Message of the last failure on this context (empty string if none).  ctx may be NULL for failures of
 * adhip_create / adhip_lower_describe (a thread-local message is returned). */
const char* adhip_last_error(adhip_ctx* ctx);

/* Device::execute -- reference src/core/ir.rs:128, src/devices/opencl/device.rs:62-88.
 * `program` is the serialised nested IR procedure (wire format: autodiff-ir-rust_amd/adhip/ir.py and
 * csrc/ir.cpp), ending in EX; `dep_ids` is the keep list (reference src/core/dependency.rs).  Starts from
 * fresh device state, uploads every CreateMat payload (host pointers inside `program` are borrowed until
 * the call returns), runs until the first EX and copies every kept id back to host memory owned by ctx.
 * The context keeps the plans and device buffers of the last few distinct programs (same command stream and
 * keep list; payload contents may differ), so executing a program again costs upload + run + read-back only;
 * ADHIP_EXEC_CACHE=0 in the environment turns that off. */
int adhip_execute(adhip_ctx* ctx, const uint8_t* program, size_t program_len, const char* const* dep_ids,
                  size_t n_dep_ids);

/* Device::get_tensor -- reference src/core/ir.rs:131, src/devices/opencl/device.rs:90-102.
 * Returns 0 and sets data/dims/ndim (memory owned by ctx, valid until the next execute/readback/destroy),
 * 1 if `id` was not kept or never defined (the reference's ValueData::none()), another code on error. */
int adhip_get_tensor(adhip_ctx* ctx, const char* id, const float** data, const uint64_t** dims, size_t* ndim);

/* Device::dot_prod_shape default -- reference src/core/ir.rs:140-142: out = {a[0], b[last]}. */
int adhip_dot_prod_shape(const uint64_t* a_dims, size_t a_ndim, const uint64_t* b_dims, size_t b_ndim, uint64_t out[2]);

/* ---- adhip_execute in stages, for callers that keep a program resident on the GPU -------------------
 * adhip_execute(ctx, ...) == program_create + program_upload + program_run + program_readback + destroy.
 * These have no separate counterpart in the reference, whose execute() does all of it in one call
 * (src/devices/opencl/device.rs:62-88). */

/* Parse, lower to kernels, compile them (hipRTC, cached per context) and allocate device buffers. */
int adhip_program_create(adhip_ctx* ctx, const uint8_t* program, size_t program_len, const char* const* dep_ids,
                         size_t n_dep_ids, adhip_program** out);
/* Copy every CreateMat payload to the device (host pointers given at create time must still be valid). */
int adhip_program_upload(adhip_program* p);
/* Run from the current device state to the first EX; returns after the stream has drained. */
int adhip_program_run(adhip_program* p);
/* The same without the final wait: the kernels are queued on the context's stream and the call returns (a loop or
 * branch that the host has to decide still waits for its predicate).  Several runs can be queued back to back;
 * adhip_program_sync waits for all of them and must be called before upload, read-back or destroy. */
int adhip_program_enqueue(adhip_program* p);
int adhip_program_sync(adhip_program* p);

/* adhip_program_enqueue for callers that cannot allocate device memory while they run (tight serving loops, harnesses
 * that forbid it; a straight-line program also under HIP stream capture).  No counterpart in the reference.
 * Every temporary of the program (partial sums of reductions, slices of split matrix products, intermediate tensors)
 * and its control-flow flags are placed in a static device array of ADHIP_STATIC_SCRATCH_BYTES that the library holds
 * on every GPU it runs on, instead of in the program's own allocations; inputs, kept tensors and ids that live across
 * control flow stay in the buffers the program got at create time.  The call makes no hipMalloc / hipFree and no
 * allocating library call, on the device or on the host, and launches every kernel directly (no graph capture or
 * instantiation, no profiling events).  A straight-line program is queued and the call returns without waiting, like
 * adhip_program_enqueue.  A program with loops or branches behaves as it does there too: the host reads predicates
 * back (a 4-byte asynchronous copy into pinned memory the context holds since adhip_create, then a wait on the
 * stream) -- once for a counted loop, once per batch of iterations for a data-dependent one, once per If -- which
 * allocates nothing but blocks, and is not legal while the caller captures the stream.  A program whose temporaries
 * and flags need more than ADHIP_STATIC_SCRATCH_BYTES is refused with an error that names both sizes.  All programs
 * of all contexts on one GPU share that GPU's array and find the last call's contents in it (every kernel writes
 * what it later reads from there, so nothing needs clearing).  Runs queued on one context follow one another on its
 * stream; runs of different contexts on the same GPU that overlap in time race on the array -- wait for one
 * (adhip_program_sync) before a run of another context starts. */
#define ADHIP_STATIC_SCRATCH_BYTES (32u << 20)
int adhip_program_enqueue_noalloc(adhip_program* p);
/* Copy kept ids to host memory owned by the context (then served by adhip_get_tensor). */
int adhip_program_readback(adhip_program* p);
void adhip_program_destroy(adhip_program* p);

/* Per-kernel timing with HIP events on the context's stream (off by default). */
int adhip_program_set_profiling(adhip_program* p, int enabled);
int adhip_program_kernel_count(adhip_program* p);
/* Launch site i: label, launches so far, total milliseconds, algorithmic bytes and flops of one launch. */
int adhip_program_kernel_stat(adhip_program* p, int i, char* label, size_t label_cap, uint64_t* launches,
                              double* total_ms, double* bytes_per_launch, double* flops_per_launch);
/* Generated HIP source of launch site i (owned by the program). */
const char* adhip_program_kernel_source(adhip_program* p, int i);
/* Text description of buffers, kernels and control structure (owned by the program). */
const char* adhip_program_describe(adhip_program* p);

/* Lower only (no GPU needed): writes the same description into `out`.  Returns non-zero and writes the
 * message into `out` on failure. */
int adhip_lower_describe(const uint8_t* program, size_t program_len, const char* const* dep_ids, size_t n_dep_ids,
                         char* out, size_t out_cap);

/* Lower and compile every generated kernel with hipRTC for `arch` (default "gfx950") without touching a
 * GPU: the build-time check that the device code is valid.  Writes a one-line summary or the error; the
 * summary ends with "; spilling kernels: <name> (<n> scalar, <n> vector registers spilled, <n> bytes of scratch
 * per lane); ..." when the compiler's metadata of a code object records any. */
int adhip_compile_check(const uint8_t* program, size_t program_len, const char* const* dep_ids, size_t n_dep_ids,
                        const char* arch, char* out, size_t out_cap);

/* ---- operators on device arrays -----------------------------------------------------------------------
 * What training and running a decoder takes beside programs: rotary positions, attention with masks, capped scores,
 * distance bias and shared heads (forward, backward, single tokens against a cache) and AdamW over many tensors.  They
 * have no counterpart in the reference.  They work on device memory that the caller holds -- the buffers of a resident
 * program (adhip_program_buffer), arrays from adhip_alloc, or any other HIP allocation on the context's device -- and
 * queue their kernels on `stream` (a hipStream_t; NULL is HIP's default stream, adhip_stream(ctx) the context's own):
 * they allocate nothing, keep nothing and do not wait, so they may be captured into a graph.  Arguments are checked
 * before anything is queued, sizes that a launch does not hold (2^32 threads) among them; what a kernel cannot check
 * (addresses) is the caller's.  Outputs must not overlap inputs except where it is said. */

enum { ADHIP_F32 = 0, ADHIP_BF16 = 1, ADHIP_I32 = 2, ADHIP_E4M3 = 3 };

/* An array in device memory: element (i0, i1, ...) is at data + sum(i * strides) elements.  Attention and rotary arrays
 * need a last stride of 1; strides may be 0 or negative on inputs only where it is said (broadcast), and an output's
 * elements must be distinct.  data = NULL: not given. */
typedef struct adhip_array {
    void* data;
    int32_t type; /* ADHIP_F32 ... */
    int32_t rank; /* 1 to 4 */
    int64_t dims[4];
    int64_t strides[4]; /* in elements */
} adhip_array;

/* Device memory of a context (freed by adhip_free or with the process, not with the context). */
int adhip_alloc(adhip_ctx* ctx, size_t bytes, void** out);
int adhip_free(adhip_ctx* ctx, void* data);
/* Copies between host and device memory on the context's stream; they return when the copy is done. */
int adhip_copy_in(adhip_ctx* ctx, void* device, const void* host, size_t bytes);
int adhip_copy_out(adhip_ctx* ctx, void* host, const void* device, size_t bytes);
/* The context's own stream (a hipStream_t), and a wait for everything queued on it. */
void* adhip_stream(adhip_ctx* ctx);
int adhip_sync(adhip_ctx* ctx);

/* The device buffer of a kept id of a resident program (dims as adhip_get_tensor gives them; dims memory is the
 * program's): where its value is after a run, and, for a CreateMat outside of loops and branches, where the next run
 * reads it from, so an operator may write there what the next run is to use.  The buffer holds packed floats and lives
 * as long as the program.  Returns 1 if `id` is not a kept id of the program. */
int adhip_program_buffer(adhip_program* p, const char* id, void** data, const uint64_t** dims, size_t* ndim);

/* Rotary positions.  x and out are [batch, length, heads, size], cos and sin f32 tables [rows, pairs] with packed rows,
 * positions int32 [batch, length]; 2 pairs <= size features of every head are turned, the others copied:
 *     (a, b) -> (a cos - b sin, a sin + b cos),   cos, sin of row positions[b, l], column i
 * with a, b the features i and i + pairs, or 2 i and 2 i + 1 where `interleaved`.  `inverse` turns the other way, which
 * is the gradient's rule.  second / second_out (data NULL: none) is another array of the same batch, length, size and
 * type that is turned by the same angles in the same launch (a step's keys beside its queries).  out may be x itself.
 * A position outside of the table gives NaN in the turned features. */
typedef struct adhip_rotary_args {
    adhip_array x, out, second, second_out;
    adhip_array cos, sin, positions;
    int32_t interleaved, inverse;
} adhip_rotary_args;
int adhip_rotary(adhip_ctx* ctx, const adhip_rotary_args* args, void* stream);

/* AdamW over many tensors: one step on each, in as few launches as their number allows.
 *     g = grad_scale gradient;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g g
 *     p = p (1 - rate decay) - rate / (1 - beta1^step) m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * in 32 bits, rounded once where p is bf16.  p and g are ADHIP_F32 or ADHIP_BF16 of `count` packed elements, m and v
 * either f32 (state_type ADHIP_F32) or ADHIP_E4M3: blocks of 256 elements, the last one padded to 256 with zeros, codes
 * [blocks, 256] and one f32 scale a block; m = code scale, sqrt(v) = code scale, scale = max(largest, 2^-100) / 448, and a
 * v that is not zero never gets the code zero.  The *_out pointers may be the inputs themselves (a step in place). */
#define ADHIP_ADAMW_BLOCK 256
typedef struct adhip_adamw_tensor {
    const void *p, *g, *m, *v;
    const float *m_scale, *v_scale; /* ADHIP_E4M3 only */
    void *p_out, *m_out, *v_out;
    float *m_scale_out, *v_scale_out;
    int64_t count;
} adhip_adamw_tensor;
typedef struct adhip_adamw_args {
    const adhip_adamw_tensor* tensors; /* host memory, read before the call returns */
    int64_t n_tensors;
    int32_t p_type, g_type, state_type;
    int32_t step; /* 1 for the first */
    double rate, beta1, beta2, eps, decay, grad_scale;
} adhip_adamw_args;
int adhip_adamw(adhip_ctx* ctx, const adhip_adamw_args* args, void* stream);
/* The same with grad_scale times the f32 number that `factor` points to in device memory when the kernels run, for instance
 * where adhip_gradient_norm left it (NULL: adhip_adamw). */
int adhip_adamw_scaled(adhip_ctx* ctx, const adhip_adamw_args* args, const float* factor, void* stream);

/* The norm over all gradients of a step, and clipping by it.
 *     norm = |grad_scale| sqrt(sum over all tensors of g g),    factor = 1 where norm <= limit, limit / norm otherwise
 * with the sum in 64 bits, added in an order that only the tensors' sizes and types decide.  norm and factor are f32 numbers in device memory
 * (factor may be NULL).  adhip_clip_gradients also writes  out = g (grad_scale factor)  of each tensor, rounded once; `out`
 * may be `g` itself; otherwise it shares memory with no gradient and no other `out`.  A gradient that is not finite shows: a NaN makes norm, factor and every clipped gradient NaN; an infinity
 * makes the norm infinite and, under a finite limit, the factor 0 (and itself NaN).  Gradients are ADHIP_F32 or ADHIP_BF16,
 * each of its own type, packed; no gradients at all have norm 0.
 * limit is above zero, and may be infinite.  workspace: adhip_gradient_norm_workspace() bytes, aligned to 8, used until the
 * call's kernels are done (only sizes and types are looked at for it). */
typedef struct adhip_gradient {
    const void* g;
    void* out; /* adhip_clip_gradients only */
    int64_t count, type;
} adhip_gradient;
typedef struct adhip_gradients_args {
    const adhip_gradient* tensors; /* host memory, read before the call returns */
    int64_t n_tensors;
    double limit, grad_scale;
    float *norm, *factor;
    void* workspace;
    size_t workspace_bytes;
} adhip_gradients_args;
int adhip_gradient_norm_workspace(adhip_ctx* ctx, const adhip_gradients_args* args, size_t* bytes);
int adhip_gradient_norm(adhip_ctx* ctx, const adhip_gradients_args* args, void* stream);
int adhip_clip_gradients(adhip_ctx* ctx, const adhip_gradients_args* args, void* stream);

/* Attention.  q and out are [batch, queries, heads, size], k and v [batch, keys, key heads, size] (f32 or bf16, one type),
 * heads a multiple of the key heads (head h reads key head h / (heads / key heads)), size at most 256.  Query i of
 * sequence b stands at position  at = i + lengths[b] - queries  (the last query at the last key), sees key j where
 *     j < lengths[b],
 *     j < prefix[b], or j <= at (causal) and, with a window, |at - j| < window,
 *     query_documents[b, i] == key_documents[b, j] >= 0 (where documents are given),
 * and scores it with
 *     z = cap tanh(scale q.k / cap) - slopes[h] |at - j|      (cap 0: scale q.k uncapped; no slopes: no second term).
 * out = softmax(z) v over what it sees, lse = log(sum(exp(z))) (f32, [batch, queries, heads]).  A query that sees nothing
 * gives out = 0 and lse = -infinity.  Keys and values behind lengths, of documents below 0, or between the prefix and the
 * beginning of the first query's window (keys up to its position - window) are not used, whatever they hold.  All others must be finite, also
 * those that no query sees for another reason (the documents of a call's queries, for instance): a tile is multiplied as a
 * whole, and a probability of zero times an infinity is NaN.  (In f32 an infinity that is seen gives NaN as well.)
 * lengths (int32 [batch]; default: keys) is clamped to 0 .. keys.  documents may lie at most 2^20 elements apart, and in f32
 * a position has at most 2^25 features over all heads.
 * workspace: device memory of at least adhip_attention_workspace() bytes, aligned to 256, used until the call's kernels
 * are done. */
typedef struct adhip_attention_args {
    adhip_array q, k, v, out, lse;
    adhip_array slopes, lengths, prefix, query_documents, key_documents; /* slopes f32 [heads], of either sign, the others int32 */
    /* backward only: gradient of out, gradients of q, k and v (of the arrays' own shapes and type) */
    adhip_array out_grad, q_grad, k_grad, v_grad;
    float scale, cap;
    int32_t causal;
    int64_t window; /* 0: none */
    void* workspace;
    size_t workspace_bytes;
} adhip_attention_args;
/* What a call on arrays of these shapes needs: only the shapes and types of q, k and v are looked at, which need not be
 * there yet. */
int adhip_attention_workspace(adhip_ctx* ctx, const adhip_attention_args* args, int backward, size_t* bytes);
int adhip_attention(adhip_ctx* ctx, const adhip_attention_args* args, void* stream);
/* Gradients of q, k and v from what adhip_attention gave (out, lse) and the gradient of out.  The order of additions
 * is fixed: the same inputs give the same bits. */
int adhip_attention_backward(adhip_ctx* ctx, const adhip_attention_args* args, void* stream);

/* Layer norm of rows.  x, added, total and out have one shape of 2 to 4 dims and one type (f32 or bf16); the last dim is the
 * row, of 1 to 16384 elements.
 *     t = x, or  total = x + added  (a sum in 32 bits, rounded as it is written) where `added` and `total` are given
 *     mean = sum(t) / size  (0 unless `centered`),  root = 1 / sqrt(sum((t - mean)^2) / size + eps)
 *     out = (t - mean) root weight + bias
 * weight and bias [size] are f32 or of x's type, both alike; no weight is a weight of 1, no bias a bias of 0.  Not centered and
 * without a bias it is RMS norm.  stats (f32, x's leading dims and 2, packed, aligned to 8 bytes; may be left out) receives mean and root.  total and out
 * may be x or added themselves, under the same strides; otherwise they share no memory with these, nor with one another. */
typedef struct adhip_layer_norm_args {
    adhip_array x, added, total, out, weight, bias, stats;
    /* backward only */
    adhip_array out_grad, total_grad, x_grad, weight_grad, bias_grad;
    double eps;
    int64_t centered;
    void* workspace; /* backward only */
    size_t workspace_bytes;
} adhip_layer_norm_args;
/* What the backward call's sums over rows need: only the shape and type of x are looked at. */
int adhip_layer_norm_workspace(adhip_ctx* ctx, const adhip_layer_norm_args* args, size_t* bytes);
int adhip_layer_norm(adhip_ctx* ctx, const adhip_layer_norm_args* args, void* stream);
/* Gradients, from x (what was normed: `total` where something was added), stats, weight and the gradient of out.  x_grad is that of t;
 * total_grad (may be left out), a gradient that reaches t by another way, is added to it.  Where something was added x_grad is the gradient of both x and
 * added.  x_grad may be out_grad, total_grad or x itself, under the same strides; otherwise it shares no memory with them.  weight_grad and bias_grad ([size], f32 or bf16, each may be left out)
 * are sums over all rows in 32 bits, added in an order that only the shape decides; with either a workspace of
 * adhip_layer_norm_workspace() bytes, aligned to 16, is used until the call's kernels are done.  The two share no memory; one array
 * given for both holds bias_grad alone.  added, total, out and bias are not looked at. */
int adhip_layer_norm_backward(adhip_ctx* ctx, const adhip_layer_norm_args* args, void* stream);

/* A gated linear recurrence over positions, each channel by itself.  x, gates and out are [batch, length, channels] (f32 or
 * bf16, one type):
 *     h[t] = a[t] h[t-1] + b[t],  out[t] = h[t],    a = sigmoid(gates), b = (1 - a) x,    or  a = gates, b = x  with `factors`
 * States are f32.  h[-1] is initial ([batch, channels]; 0 where it is not given), final receives the last state and may be
 * initial itself (a state that is carried from call to call; one position a call is a decoder's step).  lengths (int32 [batch], clamped
 * to 0 .. length): positions behind a sequence's length leave the state as it is.  documents (int32 [batch, length]): the state
 * begins at 0 at every position whose document is not that of the position before (the first position goes on from initial), and is 0 behind a
 * position of a document below 0.  Positions behind lengths or of documents below 0 give out = 0 and gradients 0, whatever x,
 * gates and out_grad hold there; everything else must be finite (gates that are no factors may be infinite).  A factor of 0 drops the state before it, whatever
 * that is.  Factors are multiplied over runs of positions: where such a product passes 2^128, results may be infinite or NaN up to the next factor of 0
 * or document.
 * states (f32 [batch, ceil(length / 256), channels]; may be left out) receives the state before every 256th position, for the
 * backward pass.  out may be x or gates themselves, under the same strides; otherwise it shares no memory with them, nor final
 * with initial.
 * Positions, where there are two and more, lie at most 2^21 elements apart.
 * workspace: adhip_recurrence_workspace() bytes, aligned to 16, used until the call's kernels are done; may be left out where that is 0. */
#define ADHIP_RECURRENCE_BLOCK 256
typedef struct adhip_recurrence_args {
    adhip_array x, gates, out, initial, final, states, lengths, documents;
    /* backward only */
    adhip_array out_grad, final_grad, x_grad, gates_grad, initial_grad;
    int64_t factors;
    void* workspace;
    size_t workspace_bytes;
} adhip_recurrence_args;
/* Only the shape and type of x are looked at; one size serves both passes, whatever `backward` is. */
int adhip_recurrence_workspace(adhip_ctx* ctx, const adhip_recurrence_args* args, int backward, size_t* bytes);
int adhip_recurrence(adhip_ctx* ctx, const adhip_recurrence_args* args, void* stream);
/* Gradients of x, gates and, where asked for, initial, from x, gates, the forward call's states, the gradient of out and, where it
 * is given, that of final ([batch, channels]); lengths, documents and factors as there.  x_grad and gates_grad may be x, gates or out_grad
 * themselves, under the same strides, and initial_grad may be final_grad itself (a gradient that is carried from call to call);
 * otherwise they share no memory with these, nor x_grad and gates_grad with one another.
 * out, initial and final are not looked at.  The order of additions is fixed. */
int adhip_recurrence_backward(adhip_ctx* ctx, const adhip_recurrence_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ADHIP_H */
