/*
 * talos_cuda.h -- C ABI of the B200 (sm_100a) decode path for Talos.
 *
 * This library replaces the Apple-Metal twin of Talos's CPU forward pass
 * (Tsuskov/talos, Rust). Each entry point names the reference interface it
 * stands in for. The Rust side binds these symbols from a `cuda` cargo feature
 * that mirrors the existing `metal` feature (Cargo.toml:28-31), with one
 * `extern "C"` declaration per entry point below.
 *
 * Conventions
 *  - Every call returns a talos_status; talos_last_error() gives the message of
 *    the last failure on the calling thread.
 *  - Host pointers everywhere unless a name ends in `_dev`; output buffers are
 *    owned by the caller.
 *  - One context drives one GPU. A context is not thread-safe: use it from one
 *    thread at a time (the reference's backend is a thread_local context,
 *    src/math/metal/mod.rs:25-29).
 *  - Calls are synchronous unless documented otherwise (the reference commits
 *    and waits once per token, src/math/metal/mod.rs:511-513).
 *  - Weights are copied to the GPU once, keyed by tensor name
 *    (src/math/metal/mod.rs:37-41,63-72), and repacked there into the
 *    GPU-friendly layouts the kernels read; the GGUF bytes are not kept.
 *  - ggml type tags: F32 = 0, Q4_0 = 2, Q8_0 = 8, Q6_K = 14
 *    (src/gguf/dtype.rs:31-41).
 */
#ifndef TALOS_CUDA_H
#define TALOS_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum talos_status {
    TALOS_OK = 0,
    TALOS_ERR_INVALID_ARG = 1, /* bad pointer, size, name, type or shape */
    TALOS_ERR_OOM = 2,         /* device or pinned-host allocation failed */
    TALOS_ERR_CUDA = 3,        /* a CUDA runtime call failed */
    TALOS_ERR_NCCL = 4,        /* an NCCL call failed */
    TALOS_ERR_TIMEOUT = 5,     /* a bounded wait ran out */
    TALOS_ERR_OOB = 6,         /* a device-side bounds check fired */
    TALOS_ERR_STATE = 7,       /* call not valid in the current state (e.g. weights missing) */
    TALOS_ERR_UNSUPPORTED = 8  /* ggml type or shape this build does not handle */
} talos_status;

enum { TALOS_F32 = 0, TALOS_Q4_0 = 2, TALOS_Q8_0 = 8, TALOS_Q6_K = 14 };
/* Further element types of the device operators' arrays (ggml tags). */
enum { TALOS_F16 = 1, TALOS_BF16 = 30 };

/* Model hyper-parameters: the fields of `Config` (src/model/config.rs:14-25) as
 * fixed-width C types (usize -> uint32_t); a binding copies them by name. */
typedef struct talos_cfg {
    uint32_t n_layer;
    uint32_t n_head;
    uint32_t n_head_kv;
    uint32_t n_embd;
    uint32_t n_ff;
    uint32_t context_length;
    uint32_t vocab_size;
    uint32_t rope_dim;
    float rms_eps;
    float rope_freq_base;
} talos_cfg;

typedef struct talos_ctx talos_ctx;
/* A packed weight on the device, for the single-matvec entry points. */
typedef struct talos_weight talos_weight;

/* Message of the last failed call on this thread ("" if none). */
const char* talos_last_error(void);

/* Number of CUDA devices visible (0 when there is no GPU). */
talos_status talos_device_count(int* out);

/* ------------------------------------------------------------ context */

/*
 * Create a decode context on CUDA device `device`. Replaces the lazily built
 * Metal context (src/math/metal/mod.rs:43-61) and `GpuKv::new`
 * (src/math/metal/mod.rs:272-281). Checks n_head_kv > 0 and
 * n_head % n_head_kv == 0 like Model::from_gguf (src/model/llama.rs:43-51).
 * The KV cache holds cfg->context_length positions.
 */
talos_status talos_ctx_create(const talos_cfg* cfg, int device, talos_ctx** out);

/*
 * Tensor-parallel context: rank `tp_rank` of `tp_size` ranks, one process per
 * GPU, joined through the 128-byte NCCL unique id that rank 0 made with
 * talos_nccl_unique_id() and shared out of band. No reference counterpart (the
 * reference is single-device); it follows the same rules as talos_ctx_create.
 */
talos_status talos_ctx_create_tp(const talos_cfg* cfg, int device, int tp_size, int tp_rank,
                                 const uint8_t* nccl_unique_id, talos_ctx** out);
talos_status talos_nccl_unique_id(uint8_t out[128]);

/*
 * Tensor parallel: the ranks of a context wait for each other inside every
 * step, each wait bounded (2 s). When any rank's step returns
 * TALOS_ERR_TIMEOUT (a rank that never launched its step, or one that stopped),
 * the ranks' barrier counters no longer agree: every rank then calls
 * talos_ctx_tp_resync while no rank has a step in flight (between two host-side
 * barriers of the caller), which waits for this rank's stream and clears its
 * counters; the next step on all ranks starts afresh. Until then every batched
 * step of a rank that saw the failure reports it again. On one GPU it only
 * clears the per-token kernel's counters. No reference counterpart.
 */
talos_status talos_ctx_tp_resync(talos_ctx* ctx);

talos_status talos_ctx_destroy(talos_ctx* ctx);

/*
 * Copy one GGUF tensor to the GPU under its GGUF name and repack it for the
 * kernels. Replaces `resident_weight` (src/math/metal/mod.rs:63-72) fed from
 * `QTensor::gpu_parts` (src/model/weights.rs:66-69). `bytes` are the raw
 * GGUF data (`len` bytes) of a row-major [rows, cols] matrix of `ggml_type`;
 * 1-D norm weights pass rows = 1. Names and shapes must be those
 * `Weights::from_gguf` binds (src/model/weights.rs:91-114). Uploading a name
 * again replaces its data. Under tensor parallelism each rank passes the FULL
 * tensor and keeps its own shard.
 */
talos_status talos_weight_upload(talos_ctx* ctx, const char* name, const void* bytes, size_t len,
                                 int ggml_type, size_t rows, size_t cols);

/*
 * How a decode step is launched. TALOS_STEP_FUSED: one persistent kernel per
 * token runs every layer, with grid-wide barriers between the phases and the
 * weight stream running on across them. TALOS_STEP_LAYERED: a graph of about
 * five kernels per layer. TALOS_STEP_AUTO (the default): FUSED when the model
 * fits it (q/k/v of a layer share a ggml type, head_dim <= 128,
 * n_embd <= 8192), else LAYERED. Both give the same results within the parity
 * bars, each bit-identical run to run. No reference counterpart (the Metal path
 * encodes one command buffer per token, src/math/metal/mod.rs:414-513).
 * talos_ctx_step_kernel reports what the next step will run (FUSED or
 * LAYERED); with FUSED requested for a model it cannot run, the next step fails
 * with TALOS_ERR_UNSUPPORTED.
 */
enum { TALOS_STEP_AUTO = 0, TALOS_STEP_FUSED = 1, TALOS_STEP_LAYERED = 2 };
talos_status talos_ctx_set_step_kernel(talos_ctx* ctx, int kind);
talos_status talos_ctx_step_kernel(talos_ctx* ctx, int* kind_out);

/* Bytes of device memory the context holds (weights + KV cache + work areas). */
talos_status talos_ctx_device_bytes(talos_ctx* ctx, size_t* out);

/*
 * The CUDA stream (cudaStream_t, as void*) every call on `ctx` runs on, so a
 * caller can time steps with CUDA events recorded on it. No reference
 * counterpart (the Metal path exposes its command queue only internally,
 * src/math/metal/mod.rs:31-34).
 */
talos_status talos_ctx_stream(talos_ctx* ctx, void** stream_out);

/*
 * Shrink the KV cache to `max_ctx` positions (never above the model's own
 * context_length) and empty it. Model::cap_context (src/model/llama.rs:69-81).
 */
talos_status talos_cap_context(talos_ctx* ctx, size_t max_ctx);

/*
 * KV cache element type: TALOS_KV_F32 (the default; the reference's KvCache
 * holds f32, src/kv_cache.rs:9-10) or TALOS_KV_F16, opt-in: K (after RoPE) and
 * V are rounded to f16 (nearest, ties to even) when appended and widened to f32
 * when read, which halves the cache's memory and its traffic per token at the
 * price of parity with the reference. Setting it reallocates and empties the
 * cache. No reference counterpart (the reference has no KV type choice).
 */
enum { TALOS_KV_F32 = 0, TALOS_KV_F16 = 1 };
talos_status talos_ctx_set_kv_dtype(talos_ctx* ctx, int dtype);
talos_status talos_ctx_kv_dtype(talos_ctx* ctx, int* dtype_out);

/*
 * Start a fresh sequence. Model::reset (src/model/llama.rs:236-238). The
 * device KV cache is indexed by position, so this only forgets the cached
 * length; positions are overwritten as they are decoded.
 */
talos_status talos_kv_reset(talos_ctx* ctx);

/* ------------------------------------------------------------ decode */

/*
 * One decode step for `token` at position `pos`; writes vocab_size logits to
 * `logits_out` (host). Model::forward_gpu (src/model/llama.rs:188-195) ->
 * math::metal::forward (src/math/metal/mod.rs:351-359). Unlike the Metal path
 * the embedding row is looked up on the GPU, so the call takes the token id.
 * Requires 0 <= pos < context length and token < vocab_size. The whole step is
 * one CUDA graph replay.
 */
talos_status talos_forward(talos_ctx* ctx, uint32_t token, size_t pos, float* logits_out);

/*
 * Like talos_forward but returns the final-norm hidden state (n_embd floats).
 * Model::forward_hidden_gpu (src/model/llama.rs:199-206) ->
 * math::metal::forward_hidden (src/math/metal/mod.rs:363-366).
 */
talos_status talos_forward_hidden(talos_ctx* ctx, uint32_t token, size_t pos, float* hidden_out);

/*
 * Greedy decode entirely on the GPU: feeds `token` at `pos`, then the argmax of
 * each step's logits at pos+1, pos+2, ... for `n` steps, and writes the n chosen
 * tokens to `tokens_out` (host). The argmax follows sample::argmax
 * (src/sample.rs:7-14): total order, last maximal index on ties. This is the
 * decode loop of src/main.rs:97-113 / benches/tokps.rs:33-41 with the logits
 * never leaving the GPU.
 */
talos_status talos_generate_greedy(talos_ctx* ctx, uint32_t token, size_t pos, size_t n,
                                   uint32_t* tokens_out);

/*
 * Feed `n` prompt tokens at positions pos0 .. pos0+n-1 (the prefill loop of
 * src/main.rs:88-95) and write the logits after the last one to `last_logits`
 * (host, may be NULL). With an f32 cache and Q4_0 / Q8_0 / Q6_K matrices the
 * prompt goes through the batched step, up to 128 consecutive positions per
 * weight pass on the tensor cores (each position attends to the ones before it,
 * as token-by-token feeding does); otherwise one token per step. Under tensor
 * parallelism every rank makes the call with the same arguments.
 */
talos_status talos_prefill(talos_ctx* ctx, const uint32_t* tokens, size_t n, size_t pos0,
                           float* last_logits);

/*
 * Batched decode: up to TALOS_MAX_BATCH independent sequences per step, each
 * with its own KV cache slot and position; every weight is read once per step
 * for all of them (a tensor-core GEMM). talos_ctx_set_batch reserves
 * `max_seqs` cache slots of the context's current context length each (0 frees
 * them; reserving empties them) for the context's model, which must have
 * Q4_0 / Q8_0 / Q6_K matrices and head_dim <= 128 (TALOS_ERR_UNSUPPORTED
 * otherwise). Under tensor parallelism every rank makes each of these calls
 * with the same arguments (talos_ctx_set_batch maps the ranks' exchange areas;
 * each step's row-parallel products are summed across ranks inside the step)
 * and every rank gets all vocab_size logits. talos_forward_batch runs one step
 * for sequences 0 .. n-1 (n <= max_seqs): sequence i feeds tokens[i] at
 * position pos[i] into slot i and gets its vocab_size logits at
 * logits_out + i * vocab_size (host). Each sequence computes what
 * Model::forward (src/model/llama.rs:85-183) computes for it alone; this is the
 * batched decode of the multi-prompt workload, which the reference runs as
 * separate token-by-token loops (src/main.rs:88-113). talos_cap_context and
 * talos_ctx_set_kv_dtype release the slots (reserve them again afterwards). No
 * reference counterpart as an entry point.
 */
#define TALOS_MAX_BATCH 64
talos_status talos_ctx_set_batch(talos_ctx* ctx, int max_seqs);
talos_status talos_forward_batch(talos_ctx* ctx, const uint32_t* tokens, const size_t* pos, int n,
                                 float* logits_out);

/*
 * The prompt of one sequence of the batch: feeds tokens[0..n) at positions
 * pos0 .. pos0+n-1 into cache slot `slot` (< max_seqs of talos_ctx_set_batch),
 * up to 128 positions per weight pass on the tensor cores, each position
 * attending to the ones before it (the prefill loop of src/main.rs:88-95 for
 * one of the multi-prompt workload's sequences); the logits after the last one
 * go to `last_logits` (host, may be NULL). Other slots are untouched.
 */
talos_status talos_prefill_slot(talos_ctx* ctx, int slot, const uint32_t* tokens, size_t n, size_t pos0,
                                float* last_logits);

/*
 * Batched greedy decode on the GPU: sequence i (slot i, i < n) feeds tokens[i]
 * at pos[i], then the argmax of its logits at pos[i]+1, ... for `steps` steps;
 * the chosen tokens go to tokens_out[k * n + i] (host, step k). The argmax is
 * sample::argmax (src/sample.rs:7-14: total order, last maximal index), taken
 * per sequence on the device, so no logits leave the GPU: talos_generate_greedy
 * for a batch, i.e. the decode loops of src/main.rs:97-113 run together.
 */
talos_status talos_generate_batch_greedy(talos_ctx* ctx, const uint32_t* tokens, const size_t* pos, int n,
                                         size_t steps, uint32_t* tokens_out);

/*
 * Batched decode with drawn tokens: as talos_generate_batch_greedy, but step k's
 * token of sequence i is talos_sample_dev's choice from its logits with settings[i]
 * and the random number u[k * n + i] (host, in [0, 1)). A temperature of 0 is the
 * greedy choice (the lowest index among equal logits, where talos_sample_dev's order
 * starts; talos_generate_batch_greedy takes the highest). The same numbers give the
 * same tokens. A row whose logits are all NaN or -inf ends the call with
 * TALOS_ERR_OOB. The reference draws one sequence's tokens on the host
 * (src/sample.rs:19-76).
 */
typedef struct talos_sampling {
    float temperature; /* <= 0: the first of the order */
    int32_t top_k;     /* 0: off */
    float top_p;       /* >= 1: off */
    float min_p;       /* 0: off */
} talos_sampling;
talos_status talos_generate_batch_sample(talos_ctx* ctx, const uint32_t* tokens, const size_t* pos, int n,
                                         size_t steps, const talos_sampling* settings, const float* u,
                                         uint32_t* tokens_out);

/*
 * A prefix shared by every sequence of the batch: positions 0 .. n-1 of slot `slot`
 * (filled before, talos_prefill_slot) become positions 0 .. n-1 of all of them. Their
 * rows are kept once, beside the slots; talos_forward_batch, talos_prefill_slot and the
 * batched generation then attend to them once for all sequences (the tensor-core
 * attention of talos_attention_shared_dev) and to the slots' own rows from position n
 * on, and refuse positions below n. The slots keep rows by their absolute positions.
 * A call with a prefix in place extends it from the slot's rows behind it, or cuts it.
 * The slot is then the one that the prefix came from, or one whose sequence went on
 * behind it (to extend it, up to the last of its positions); a slot that holds another
 * prompt, or whose rows are older than the sharing, is refused (INVALID_ARG): end the
 * sharing first. n = 0 ends it, whatever the slot (the slots' rows below the old prefix
 * are then what they were before it, so only slots that were filled themselves can go
 * on). Takes the memory of
 * one more slot, from the first call to the release of the slots. The attention's
 * scores and weights are exact to about 22 bits, like the f32 path's own roundings;
 * results with and without sharing differ in their last bits. It pays from some hundred
 * shared rows on: behind a prefix of 64 rows a step was up to 11 % slower with it. Under tensor parallelism
 * every rank makes the call. No reference counterpart.
 */
talos_status talos_batch_share(talos_ctx* ctx, int slot, size_t n);

/*
 * Copies of rows between the batch's cache slots, all at once (talos_kv_move_dev on the
 * context's cache): the rows of positions start .. start+len-1 of slot src, in every
 * layer, to slot dst. A prompt forked into other slots, live sequences moved to the
 * front (decode steps take slots 0 .. n-1), or slots exchanged; every source is read as
 * it was before the call, no slot may be the destination of two copies. Under tensor
 * parallelism every rank makes the call. No reference counterpart.
 */
typedef struct talos_kv_copy {
    uint32_t src, dst, start, len;
} talos_kv_copy;
talos_status talos_batch_move(talos_ctx* ctx, const talos_kv_copy* moves, size_t n);

/*
 * Teacher-forced perplexity of tokens[0..n) (n >= 2): eval::perplexity
 * (src/eval.rs:35-52). The tokens are scored in chunks of the context length,
 * each from an empty KV cache; at each position the negative log-likelihood of
 * the next token (token_nll, src/eval.rs:18-23: log-sum-exp in f64) is added on
 * the GPU, so no logits leave the device (up to 128 positions per weight
 * pass where talos_prefill takes its batched steps). Writes exp(mean NLL) to *ppl_out and,
 * if not NULL, the NLL sum and the number of scored positions. Leaves the KV
 * cache holding the last chunk.
 */
talos_status talos_perplexity(talos_ctx* ctx, const uint32_t* tokens, size_t n, float* ppl_out,
                              double* nll_sum_out, size_t* scored_out);

/*
 * Run one decode step (as talos_forward, logits stay on the GPU) and add the
 * device time in milliseconds of each part of it into kernel_ms[kind] and the
 * number of such parts into launches[kind] (either may be NULL), kind =
 * talos_kernel_kind. LAYERED steps launch their kernels one by one with CUDA
 * events between them. FUSED steps run the per-token kernel once with phase
 * time stamps (the device's global timer, read by CTA 0 as it passes each
 * grid barrier); the last phase also carries the launch and drain time. For
 * benchmarks. No reference counterpart.
 */
enum talos_kernel_kind {
    TALOS_K_EMBED = 0,  /* token embedding row dequant */
    TALOS_K_QKV = 1,    /* RMSNorm + q/k/v matvec + RoPE + KV append */
    TALOS_K_ATTN = 2,   /* split-position GQA attention */
    TALOS_K_OPROJ = 3,  /* attn_output matvec + residual */
    TALOS_K_GATEUP = 4, /* RMSNorm + gate/up matvec + SwiGLU */
    TALOS_K_DOWN = 5,   /* ffn_down matvec + residual */
    TALOS_K_OUTPUT = 6, /* final RMSNorm + output matvec (+ argmax) */
    TALOS_K_COUNT = 7
};
talos_status talos_profile_step(talos_ctx* ctx, uint32_t token, size_t pos, double* kernel_ms,
                                uint32_t* launches);

/*
 * Run one decode step of the per-token kernel with profiling stamps and copy
 * them to `out` (host): for phase p (in step order: per layer q/k/v,
 * attention, o-proj, gate/up, down; then the output phase) and CTA c, four
 * device global-timer values in ns at out[(p * n_cta + c) * 4 + k]: k = 0 the
 * CTA entered the phase, 1 its inputs were staged, 2 its compute finished,
 * 3 it arrived at the phase's barrier (0 where a stamp does not apply). `cap`
 * is the length of `out` in elements; *n_phase and *n_cta receive the
 * dimensions. TALOS_ERR_UNSUPPORTED when steps run the layered graph. For
 * benchmarks; no reference counterpart.
 */
talos_status talos_profile_phases(talos_ctx* ctx, uint32_t token, size_t pos, uint64_t* out, size_t cap,
                                  int* n_phase, int* n_cta);

/* ------------------------------------------------------------ kernels */

/*
 * Dequantize n_elems values of `ggml_type` from raw GGUF `bytes` (host) into
 * `out` (host) on the GPU, bit-exact with GgmlType::dequantize
 * (src/gguf/dtype.rs:64-121). Test hook for the bit-exact contract.
 */
talos_status talos_dequant(int ggml_type, const void* bytes, size_t n_elems, float* out);

/*
 * Greedy choice over n logits (host) on the current CUDA device:
 * sample::argmax (src/sample.rs:7-14), the maximum under f32::total_cmp
 * (-NaN < -inf < ... < -0.0 < +0.0 < ... < +inf < +NaN) and the LAST maximal
 * index on ties. The decode step's own argmax (talos_generate_greedy, the
 * logits epilogue) uses the same key. n must be 1 .. 2^32-1 (the reference
 * panics on empty logits).
 */
talos_status talos_argmax(const float* logits, size_t n, uint32_t* index_out);

/*
 * One fused dequant-matvec y = W x on device `device`, with W uploaded for this
 * call only. math::metal::matvec_f32 / matvec_quant
 * (src/math/metal/mod.rs:195-225). x: cols floats, y: rows floats (host).
 */
talos_status talos_matvec(int device, int ggml_type, const void* bytes, size_t len, size_t rows,
                          size_t cols, const float* x, float* y);

/*
 * Matvec against a weight kept on the GPU under `name` in `ctx`: uploaded on
 * first use and reused while the byte length stays the same, even if the bytes
 * differ. math::metal::matvec_f32_resident / matvec_quant_resident
 * (src/math/metal/mod.rs:227-253), with the cache rule of
 * src/math/metal/mod.rs:63-72.
 */
talos_status talos_matvec_resident(talos_ctx* ctx, const char* name, int ggml_type,
                                   const void* bytes, size_t len, size_t rows, size_t cols,
                                   const float* x, float* y);

/*
 * Device-level matvec for benchmarks: pack a weight onto device `device` once,
 * then run y_dev = W x_dev on a CUDA stream (cudaStream_t passed as void*,
 * NULL = legacy default stream) without synchronizing. x_dev/y_dev are device
 * pointers of cols / rows floats. No reference counterpart; it exposes the
 * kernel that QTensor::matvec (src/model/weights.rs:47-55) becomes.
 */
talos_status talos_weight_create(int device, int ggml_type, const void* bytes, size_t len,
                                 size_t rows, size_t cols, talos_weight** out);
talos_status talos_weight_destroy(talos_weight* w);
talos_status talos_weight_packed_bytes(const talos_weight* w, size_t* out);
talos_status talos_matvec_dev(const talos_weight* w, const float* x_dev, float* y_dev,
                              void* stream);

/*
 * talos_matvec_dev without allocating: a split-K variant (each CTA takes one
 * 16-row tile and one slice of the columns; the slices' partial sums meet in a
 * fixed-size scratch array that the library holds as static device memory, and
 * the last slice of a tile adds them in slice order). For callers that must not
 * allocate device memory during decoding: a runtime that reserves the device's
 * memory up front, or a loop that cannot take the device-wide synchronisation
 * of cudaMalloc / cudaFree. Limits: at most 65,536 rows (the scratch is 2 MB of
 * partial sums + 16 KB of arrival counters) and columns whose staged input
 * fits shared memory (about 47,000); larger weights fail with
 * TALOS_ERR_UNSUPPORTED. The first call on a device resolves the scratch's
 * address (cudaGetSymbolAddress); make it before any stream capture. Calls
 * share the scratch: two calls in flight at once (other streams, other
 * threads) race, so serialise them. Results agree with talos_matvec_dev to
 * rounding (another summation order) and are identical call to call. Every
 * device wait is bounded (2 s): a 16-row tile any of whose K slices gave up
 * waiting for its weight copy comes out as 16 NaN rows (the call itself still
 * returns TALOS_OK, since it does not synchronise). No reference counterpart.
 */
talos_status talos_matvec_dev_noalloc(const talos_weight* w, const float* x_dev, float* y_dev, void* stream);

/*
 * Benchmark helper: capture `reps` back-to-back talos_matvec_dev launches that
 * cycle through the n weights ws[0..n-1] (same shape) into one CUDA graph, replay
 * it once to warm up and once timed with CUDA events, and write the average
 * device microseconds per launch to *us_per_launch. Host launch overhead is not
 * in the number. No reference counterpart.
 */
talos_status talos_matvec_bench(const talos_weight* const* ws, int n, const float* x_dev,
                                float* y_dev, int reps, float* us_per_launch);

/* ------------------------------------------------------------ batch operators
 *
 * Device operators for many sequences that start from one prompt. Pointers named
 * *_dev and those inside the argument structs' "device" fields are device
 * pointers on CUDA device `device`; the work is enqueued on `stream`
 * (cudaStream_t as void*, NULL = legacy default stream) and not waited for, the
 * caller's current device is left as it was, nothing is allocated, and the calls
 * can be captured into a CUDA graph.
 */

/*
 * The choice of a token per row of logits, with one given random number each:
 * sample (src/sample.rs:19-76) on the GPU, with min-p besides. In the order of
 * descending logit (equal logits: the lower index first):
 *   w_i = exp((logit_i - max) / temperature)
 *   top_k > 0:  keep the first top_k                          (0: all)
 *   top_p < 1:  of these the shortest prefix with weight >= top_p * their weight
 *               (at least one; >= 1: all)
 *   min_p > 0:  of these the ones with w_i >= min_p (min_p above 1 acts as 1)
 *   the token is the first whose cumulative weight exceeds u * (kept weight).
 * temperature <= 0 (or NaN) takes the first of the order, as top_k = 1 does:
 * where several logits are exactly equal, talos_argmax takes the last index and
 * this the first. NaN logits count as -inf; -inf is never chosen, and +inf
 * shares the whole weight with the other +inf. A row with nothing above -inf
 * gives token -1 and probability 0. u outside [0, 1) is clamped (NaN: 0).
 * Weights are exact to 2^-42 of the largest one and their sums do not depend on any order,
 * so a call gives the same tokens every time. probs (optional): the weight of
 * the token over the kept weight.
 */
typedef struct talos_sample_args {
    int device;
    int type;            /* TALOS_F32, TALOS_F16 or TALOS_BF16 */
    uint32_t n, vocab;   /* rows; logits per row, 1 .. 1,048,576 */
    const void* logits;  /* device, [n] rows */
    size_t row_stride;   /* elements between rows, >= vocab if n > 1 */
    const float* u;      /* device, [n] */
    /* device, [n] each, or NULL: the value below for every row */
    const float* temperature_dev;
    const int32_t* top_k_dev;
    const float* top_p_dev;
    const float* min_p_dev;
    float temperature;
    int32_t top_k;
    float top_p;
    float min_p;
    int32_t* tokens; /* device, [n] */
    float* probs;    /* device, [n], or NULL */
} talos_sample_args;
talos_status talos_sample_dev(const talos_sample_args* args, void* stream);

/*
 * The same for one row of n host logits on the current CUDA device, beside
 * talos_argmax: *index_out is the token; prob_out may be NULL. A row with
 * nothing above -inf fails with TALOS_ERR_INVALID_ARG.
 */
talos_status talos_sample(const float* logits, size_t n, float u, float temperature, int32_t top_k, float top_p,
                          float min_p, uint32_t* index_out, float* prob_out);

/*
 * Attention of n sequences over one shared prefix and a suffix of each one's own
 * (a prompt that many sequences continue): for sequence i and query head h, with
 * kv head h / (n_head / n_head_kv), the keys are prefix rows 0 .. prefix_len-1
 * and rows 0 .. lens[i]-1 of cache slot slots[i];
 *   out[i][h] = softmax(scale * q . K) V        (src/model/llama.rs:135-155)
 * and zeros where there is no key at all, or none whose score in f32 is above -inf
 * (such a key has no weight beside others). The prefix is read once for all
 * sequences of a row tile (128 / (n_head / n_head_kv) of them) instead of once
 * per sequence. What lies behind lens[i] changes nothing (the rest of a tile of a
 * named slot may be read along); slots that no sequence names are not read. Types (q and out, cache): F32 with F32 (the reference's cache) or F16,
 * F16 with F16, BF16 with BF16; f32 queries get f32 accuracy on the tensor
 * cores. head_dim up to 128, a multiple of 8 (4 where all is F32); n_head at
 * most 128 times n_head_kv; n up to 1024. UNSUPPORTED beyond 2^30 tiles of 64 keys (of
 * one row tile over the kv heads, or of one kv head over the row tiles). The last
 * dimension is contiguous; strides are in elements; pointers and strides are multiples
 * of 16 bytes. K and V share their strides. lens are clamped to 0 .. slot_len; a
 * sequence whose slot is out of range has no suffix. Keys that are attended to hold
 * finite values; an infinite or NaN value makes its own dimension of the outputs that
 * attend to it infinite or NaN. What a sequence's own rows hold does not reach another's
 * output.
 *
 * work: talos_attention_shared_work bytes of device memory, 16-byte aligned,
 * used by this call alone until it has run (two calls in flight, or two graphs
 * that may run at once, need one each); its contents need not be kept or set.
 * Every wait inside is bounded (a number of polls, seconds at most): rows of a CTA whose
 * wait ran out are NaN. f32 accuracy: q keeps 22 bits per element (of its row's largest
 * element), the weights 22 bits, an element of an f32 cache 22 bits or 2^-39 of the
 * largest element among the 64 rows of its tile. 16-bit types: the weights are rounded
 * to the type (half a step of 2^-11 or 2^-8 each) and summed as rounded, the rest is f32
 * (the tensor core's sums of 16 tiles at a time lose about 1.5e-5 of themselves). An output
 * has therefore 1.3 to 1.4 times the error of one from unrounded weights.
 * No reference counterpart (the reference decodes one sequence at a time).
 */
typedef struct talos_attention_shared_args {
    int device;
    int q_type, kv_type;
    uint32_t n, n_head, n_head_kv, head_dim;
    uint32_t prefix_len;          /* may be 0 */
    uint32_t n_slots, slot_len;   /* the caches' slots and rows per slot */
    const void* q;                /* device, [n][n_head][head_dim] */
    size_t q_stride_n, q_stride_h;
    const void *k_prefix, *v_prefix; /* device, [prefix_len][n_head_kv][head_dim] */
    size_t prefix_stride_t, prefix_stride_h;
    const void *k, *v;            /* device, [n_slots][slot_len][n_head_kv][head_dim] */
    size_t slot_stride, slot_stride_t, slot_stride_h;
    const int32_t* slots;         /* device, [n], or NULL: sequence i in slot i */
    const int32_t* lens;          /* device, [n] */
    void* out;                    /* device, [n][n_head][head_dim] */
    size_t out_stride_n, out_stride_h;
    float scale;                  /* usually 1 / sqrt(head_dim); 1e-30 .. 1e30 */
} talos_attention_shared_args;
talos_status talos_attention_shared_work(int device, uint32_t n, uint32_t n_head, uint32_t n_head_kv, size_t* out);
talos_status talos_attention_shared_dev(const talos_attention_shared_args* args, void* work, size_t work_bytes,
                                        void* stream);

/*
 * Move rows between cache slots: for every i, rows [start, start + len) of slot
 * src become those rows of slot dst, in each of the n_base arrays (K and V,
 * say) and each of the n_outer planes (layers). The moves are simultaneous:
 * every one reads what the slots held before the call, whatever the order
 * (compaction, permutations, one slot to many). Rows outside the ranges keep
 * their values. A slot may be the destination of one move only (INVALID_ARG
 * otherwise); src == dst or len == 0 does nothing. At most 512 moves. The
 * geometry must not make rows overlap, within an array or between two (INVALID_ARG;
 * interleaved arrays are fine). No reference counterpart
 * (the reference keeps one sequence, src/kv_cache.rs:7-52).
 */
typedef struct talos_kv_slots {
    int device;
    int n_base;         /* arrays, 1 .. 8 */
    void* const* base;  /* host array of device pointers */
    uint32_t n_slots, n_outer, n_rows;
    size_t slot_stride, outer_stride, row_stride; /* bytes */
    size_t row_bytes;
} talos_kv_slots;
talos_status talos_kv_move_dev(const talos_kv_slots* slots, const talos_kv_copy* moves, size_t n, void* stream);

#ifdef __cplusplus
}
#endif
#endif
