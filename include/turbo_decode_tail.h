/*
 * turbo_decode_tail.h -- C ABI of the MI355X (gfx950) decode tail.
 *
 * Replaces the decode tail of ForwardRunner::produce_token (src/runner.cpp:719-807):
 *
 *   final RMSNorm -> affine-int4 tied LM head (group 64, BF16 scale + bias) over the whole
 *   vocabulary -> final-logit softcap -> logit modifiers -> greedy argmax or sampled draw
 *
 * Conventions follow include/gturbo/c_api.h:
 *   - plain C types and pointers only; every entry point catches all C++ exceptions;
 *   - handle-returning calls return NULL on failure, int-returning calls return 1 on success
 *     and 0 on failure; the reason is in turbo_lmhead_last_error() (thread-local, "" after a
 *     successful call, valid until the next failing call on the same thread; c_api.h:74-78);
 *   - option structs must be initialised by their *_default() function before use, because
 *     zero-initialisation is not valid (c_api.h:30-47).
 *
 * Memory: unless a comment says "host", every buffer pointer is a HIP device pointer. All
 * work is enqueued on the handle's stream (turbo_lmhead_set_stream; default: the null stream)
 * and is asynchronous to the host. One step in flight per handle; calls on one handle must be
 * serialised by the caller, as the reference serialises generation (README.md:202-206).
 */
#ifndef TURBO_DECODE_TAIL_H
#define TURBO_DECODE_TAIL_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TURBO_DT_API __attribute__((visibility("default")))

/* ---- ABI version ------------------------------------------------------------------------- */

/*
 * No counterpart in the reference (its C API has one struct, checked by turbo_options_default).
 * TURBO_DT_ABI_VERSION changes whenever a struct layout or an entry point's meaning changes.
 * A caller compiled against this header checks, once at load time, that
 * turbo_abi_version() == TURBO_DT_ABI_VERSION and that turbo_abi_struct_size() agrees with its
 * sizeof for every struct it passes; a library of another layout would otherwise read or write
 * past the caller's arrays (TurboRowReport per row, for example) without any error.
 */
#define TURBO_DT_ABI_VERSION 1u
enum {
    TURBO_ABI_LMHEAD_DESC = 0,    /* TurboLMHeadDesc */
    TURBO_ABI_BUNDLE_TENSOR = 1,  /* TurboBundleTensor */
    TURBO_ABI_SAMPLING_ROW = 2,   /* TurboSamplingRow */
    TURBO_ABI_STEP_INPUTS = 3,    /* TurboStepInputs */
    TURBO_ABI_ROW_REPORT = 4,     /* TurboRowReport */
    TURBO_ABI_STEP_OUTPUTS = 5,   /* TurboStepOutputs */
    TURBO_ABI_KV_CACHE_DESC = 6,  /* TurboKvCacheDesc */
    TURBO_ABI_ROTARY_DESC = 7,    /* TurboRotaryDesc */
    TURBO_ABI_QKV_INPUTS = 8,     /* TurboQkvInputs */
    TURBO_ABI_ATTENTION_INPUTS = 9, /* TurboAttentionInputs */
    TURBO_ABI_BATCH_PLAN = 10,    /* TurboBatchPlan */
    TURBO_ABI_PAGES_RELEASE = 11, /* TurboPagesRelease */
    TURBO_ABI_TREE_ACCEPT = 12,   /* TurboTreeAccept */
    TURBO_ABI_PROMPT_INPUTS = 13  /* TurboPromptInputs */
};
TURBO_DT_API uint32_t turbo_abi_version(void);
/* sizeof of the struct TURBO_ABI_* names, as the library was built; 0 for an unknown id. */
TURBO_DT_API size_t turbo_abi_struct_size(int which);

/* ---- errors ------------------------------------------------------------------------------ */

/* Replaces turbo_engine_last_error (include/gturbo/c_api.h:74-78; src/c_api.cpp:29-40). */
TURBO_DT_API const char* turbo_lmhead_last_error(void);

/* ---- head creation ----------------------------------------------------------------------- */

/*
 * Describes the tied LM head and final norm. Field meanings follow the manifest constants
 * (include/gturbo/manifest.hpp:23-50) and the resident-table layout the reference uploads at
 * ForwardRunner::initialize (src/runner.cpp:260-292, :324-357):
 *   weight       [vocab][hidden/2] bytes, element c in byte c/2, low nibble when c is even
 *                (docs/GTURBO_FORMAT.md:40; shaders/Common.hlsli:27-29)
 *   scales       [vocab][hidden/64] BF16, row-major
 *   biases       [vocab][hidden/64] BF16, row-major; dequantised w = q * scale + bias
 *   norm_weight  [hidden] BF16 model.norm.weight, applied as plain w (not 1 + w,
 *                src/cpu_reference.cpp:40-42); NULL means no weight
 */
typedef struct {
    uint32_t vocab_size;        /* 262144 for Gemma 4 (manifest.hpp:32) */
    uint32_t hidden_size;       /* 2816 (manifest.hpp:24); must be a multiple of 64 */
    uint32_t group_size;        /* must be 64 (src/cpu_reference.cpp:32) */
    float final_logit_softcap;  /* 30 (manifest.hpp:34); <= 0 disables the softcap */
    float rms_norm_eps;         /* 1e-6 (manifest.hpp:39) */
    int weights_on_device;      /* 0: the four pointers are host memory; 1: device memory */
    const uint8_t* weight;
    const uint16_t* scales;
    const uint16_t* biases;
    const uint16_t* norm_weight;
    int device;                 /* HIP device ordinal */
} TurboLMHeadDesc;

/*
 * ---- .gturbo bundle: resident.bin ---------------------------------------------------------
 * One tensor of the resident index (include/gturbo/resident_index.hpp:17-27), with the
 * quantisation geometry the reference derives from it (src/cpu_reference.cpp:229-247).
 */
typedef struct {
    uint32_t dtype;             /* 0 U32 (packed quantised words), 1 BF16, 2 FP16, 3 FP32 */
    uint32_t shape[4];
    uint64_t file_offset, size_bytes;
    uint64_t scale_offset, scale_size;  /* scale_size 0: not quantised */
    uint64_t bias_offset, bias_size;
    uint32_t quantized;
    uint32_t rows;              /* shape[0]; 1 for an empty shape */
    uint32_t in_dim;            /* quantised: scale_size / 2 / rows * 64; otherwise rows */
    uint32_t bits;              /* quantised: 4 when shape[1] * 8 == in_dim, else 8; otherwise 16 */
} TurboBundleTensor;

/* Decodes the 24-byte resident header (ResidentIndexCodec::decode_header,
 * src/resident_index.cpp:42-52): out = {index_size, resident_size, entry_count}. 1/0. */
TURBO_DT_API int turbo_bundle_decode_header(const uint8_t* bytes, size_t count, uint64_t out[3]);
/* Reads and validates the index region of the resident.bin at path
 * (ResidentIndexCodec::decode_region, src/resident_index.cpp:54-104) and describes tensor
 * `name` (ForwardRunner::resident_ref, src/runner.cpp:324-347). 1/0. */
TURBO_DT_API int turbo_bundle_find_tensor(const char* resident_path, const char* name,
                                          TurboBundleTensor* out);
/*
 * Creates the head from a bundle's resident.bin: model.embed_tokens.weight (the tied table,
 * 4-bit, one index entry with its scale and bias regions) and model.norm.weight (BF16), read
 * from their 16 KB-aligned regions (docs/GTURBO_FORMAT.md:26-58). The softcap and eps are the
 * manifest's arch.final_logit_softcap and arch.rms_norm_eps (include/gturbo/manifest.hpp:34,
 * :39), passed by the caller that parsed manifest.json. Replaces the runner's resident lookups
 * for this path (src/runner.cpp:324-357, :722-723, :773). NULL on failure.
 */
TURBO_DT_API void* turbo_lmhead_create_from_bundle(const char* resident_path, float final_logit_softcap,
                                                   float rms_norm_eps, int device);

/* Fills the Gemma 4 26B-A4B constants; the four pointers are NULL. */
TURBO_DT_API void turbo_lmhead_desc_default(TurboLMHeadDesc* out);

/*
 * Copies the table into HBM in the kernels' tiled layout (the caller's buffers may be freed
 * afterwards) and allocates per-step scratch. Replaces the resident upload and buffer set-up
 * of ForwardRunner::initialize for this path (src/runner.cpp:211-215, :260-292).
 * Returns NULL on failure. Batches above two rows compute on the matrix cores in fp16: a table
 * with a scale or bias of magnitude above 65504 is accepted, but such calls on it then fail with
 * an error (one- and two-row calls are unaffected). Hidden states have no such limit.
 */
TURBO_DT_API void* turbo_lmhead_create(const TurboLMHeadDesc* desc);
/* Waits for the handle's stream (the one set by turbo_lmhead_set_stream, which must still exist;
 * other streams are not waited for) and frees everything (src/runner.cpp:25-42). NULL is a
 * no-op. */
TURBO_DT_API void turbo_lmhead_destroy(void* handle);
/* hip_stream is a hipStream_t (NULL = the null stream). Must be created at default priority.
 * Switching to another stream first waits for the current one, whose steps may still be using
 * the handle's scratch buffers. */
TURBO_DT_API int turbo_lmhead_set_stream(void* handle, void* hip_stream);
/* Waits for the handle's stream. Returns 0 (once) when a step since the last call found a full
 * history under TURBO_STEP_APPEND_HISTORY (TURBO_STATUS_HISTORY_FULL). */
TURBO_DT_API int turbo_lmhead_synchronize(void* handle);
/* Largest batch one step accepts, and the largest bias_stride (logit-bias entries per row).
 * History length is not limited. */
TURBO_DT_API int turbo_lmhead_limits(void* handle, int* max_batch, int* max_row_modifiers);

/* ---- sampling parameters ----------------------------------------------------------------- */

enum {
    TURBO_RNG_PHILOX = 0,    /* u = Philox4x32-10(key = seed, counter = counter), 24-bit */
    TURBO_RNG_REFERENCE = 1  /* u = next_uniform(seed_for(has_seed, seed, position = counter)),
                                the reference's map (src/sampling.cpp:18-28, :63-72) */
};

enum {
    /* Lifts the reference's 256-candidate shortlist and accepts top_k == 0 with top_p < 1:
     * nucleus over the full vocabulary, as the full-sort sampler of
     * tests/test_sampling.cpp:36-84. Without it the semantics are exactly sample_token's. */
    TURBO_ROW_FULL_VOCAB = 1u
};

/*
 * Per-row sampling parameters. The first four fields are SamplingParams
 * (include/gturbo/sampling.hpp:21-30); the rest are extensions.
 */
typedef struct {
    float temperature;          /* 0 = greedy */
    float top_p;                /* (0, 1]; 1 = no nucleus */
    int top_k;                  /* 0..256; 0 = off */
    float repetition_penalty;   /* > 0; 1 = off; applied per history occurrence */
    float presence_penalty;     /* extension: l -= presence for ids seen at least once */
    float frequency_penalty;    /* extension: l -= frequency * count */
    int rng;                    /* TURBO_RNG_* */
    int has_seed;               /* TURBO_RNG_REFERENCE only */
    uint64_t seed;
    uint64_t counter;           /* Philox counter (decode step), or the reference's int position
                                   (two's complement; must fit in int for TURBO_RNG_REFERENCE) */
    uint32_t flags;             /* TURBO_ROW_* */
} TurboSamplingRow;

/* Greedy, no penalties, Philox with seed 0 counter 0 (sampling.hpp:21-30 defaults). */
TURBO_DT_API void turbo_sampling_row_default(TurboSamplingRow* out);
/* validate_sampling (src/sampling.cpp:32-54). Returns 1 if valid; else 0 and the reason. */
TURBO_DT_API int turbo_validate_sampling(const TurboSamplingRow* row);
/* splitmix64 and seed_for (src/sampling.cpp:56-72). */
TURBO_DT_API uint64_t turbo_splitmix64(uint64_t x);
TURBO_DT_API uint64_t turbo_seed_for(int has_seed, uint64_t seed, int position);
/* The uniform a step draws for this row (host computation of the device's value). */
TURBO_DT_API float turbo_row_uniform(const TurboSamplingRow* row);

/* ---- the decode-tail step ---------------------------------------------------------------- */

enum { TURBO_HIDDEN_F32 = 0, TURBO_HIDDEN_BF16 = 1 };

enum {
    TURBO_STEP_NORMED = 1u,          /* hidden is already normalised: skip the final RMSNorm */
    TURBO_STEP_APPEND_HISTORY = 2u   /* append each row's token to its history on the device
                                        (src/runner.cpp:878), incrementing history_len. The
                                        reference's history grows without bound; here it holds
                                        history_stride ids per row, so the caller sizes the
                                        stride for the initial length plus every step it will
                                        run. A row whose history is full keeps its token but
                                        does not append it: its report has
                                        TURBO_STATUS_HISTORY_FULL and the next
                                        turbo_lmhead_synchronize returns 0 with the reason. */
};

/* Row-strided side inputs. Any group may be NULL / zero to disable it. */
typedef struct {
    int batch;                  /* 1 .. max_batch */
    const void* hidden;         /* [batch][hidden_size], TURBO_HIDDEN_* (buf_hidden_ at :722) */
    int hidden_dtype;
    uint32_t flags;             /* TURBO_STEP_* */
    const TurboSamplingRow* rows; /* HOST array [batch], copied by the call */
    /* history ids (src/runner.cpp:801-803): row b has history_len[b] ids at
     * history + b * history_stride; ids >= vocab are ignored (src/sampling.cpp:82). */
    uint32_t* history;
    uint32_t history_stride;
    uint32_t* history_len;
    /* banned-token bitmask (extension): bit (id % 32) of word ban_bits[b * ban_stride + id/32] */
    const uint32_t* ban_bits;
    uint32_t ban_stride;
    /* sparse logit bias (extension): bias_count[b] pairs at b * bias_stride */
    const uint32_t* bias_ids;
    const float* bias_values;
    uint32_t bias_stride;
    const uint32_t* bias_count;
    /* injected uniforms [batch] in [0, 1); NULL = derive from each row's rng */
    const float* uniforms;
} TurboStepInputs;

/* Diagnostics per row (optional). */
typedef struct {
    float max_logit;        /* row maximum after modifiers */
    float u;                /* uniform used */
    uint32_t shortlist;     /* candidate list size (want) */
    uint32_t cut;           /* survivors after top-p / top-k */
    uint32_t rank;          /* token's position among the survivors */
    uint32_t path;          /* 0 greedy, 1 shortlist, 2 full-vocabulary value bins,
                               3 degenerate, 4 radix fallback (massive ties) */
    double total;           /* sum exp(l - max) over the row */
    double denom;           /* survivor weight sum */
    double r;               /* u * denom */
    uint32_t status;        /* TURBO_STATUS_* bits */
    uint32_t reserved;
} TurboRowReport;

enum {
    /* TURBO_STEP_APPEND_HISTORY found history_len == history_stride: the token was returned but
     * not appended. turbo_lmhead_synchronize then fails (once) with the row in the message. */
    TURBO_STATUS_HISTORY_FULL = 1u
};

typedef struct {
    uint32_t* tokens;        /* [batch]; 0xFFFFFFFF marks a degenerate distribution */
    float* logits;           /* optional [batch][vocab]: final logits after all modifiers */
    TurboRowReport* report;  /* optional [batch] */
} TurboStepOutputs;

/*
 * One decode-tail step for a batch of independent rows: (RMSNorm) -> int4 head -> softcap ->
 * bias -> repetition -> presence/frequency -> ban -> greedy or sampled token per row.
 * Replaces src/runner.cpp:719-807 (RMSNormK, LMHeadGreedy + ArgmaxReduce or GemvInt4 x5 +
 * Softcap + readback + apply_repetition_penalty + sample_token). Every row is validated
 * first (turbo_validate_sampling); an invalid row fails the call before anything is enqueued.
 *
 * A row's logits never depend on the other rows' values. Their last bits follow the kernel that the
 * vocabulary and the batch size choose (here and in turbo_lmhead_logits): the same for one and two
 * rows, and the same for every batch of three and more rows, except over 8,193 to 49,152 ids (129 to
 * 768 tiles of 64), where the batches with tiles x ceil(batch / 32) <= 1024 share one set of bits
 * and the larger ones another.
 */
TURBO_DT_API int turbo_lmhead_step(void* handle, const TurboStepInputs* in,
                                   const TurboStepOutputs* out);

/*
 * Affine-int4 matrix-vector product, out[b][r] = sum_c (q[r][c] * scale + bias) * x[b][c], at
 * any shape a head accepts (rows up to 2^24, in_dim a multiple of 64 up to 8192): the
 * reference's GemvInt4 (shaders/GemvInt4.hlsl:1-38) as dispatched for the q/k/v/o projections,
 * the shared expert and the routed experts (src/runner.cpp:431-442, :621-646, :671-678). A
 * matrix is a handle created with vocab_size = rows, hidden_size = in_dim, final_logit_softcap
 * 0 and no norm weight. x: [batch][in_dim] (TURBO_HIDDEN_*), out: [batch][rows] FP32, device.
 */
TURBO_DT_API int turbo_int4_matvec(void* handle, const void* x, int x_dtype, int batch, float* out);

/*
 * ---- int4 matrices of the layer loop ------------------------------------------------------
 * A matrix handle holds one affine-int4 weight matrix (rows x in_dim, group 64, BF16 scale +
 * bias; the reference layout of turbo_lmhead_create) in the kernels' tiled layout and nothing
 * else, so its device footprint is the table's size (rows * in_dim / 2 + rows * in_dim / 16
 * bytes). These replace the GemvInt4 dispatches of the layer loop (shaders/GemvInt4.hlsl:1-38;
 * src/runner.cpp:431-442, :612-646, :671-678) for the expert slots and projections.
 */
/* rows 1..16777216, in_dim a multiple of 64 up to 8192. Allocates the table only; the contents
 * are undefined until turbo_int4_matrix_load. NULL on failure. */
TURBO_DT_API void* turbo_int4_matrix_create(uint32_t rows, uint32_t in_dim, int device);
/* Repacks one matrix into the handle (the expert streamer's slot refill, src/streamer.cpp:171-214).
 * weights_on_device = 1: the three pointers are device memory (for example the slot's buffer at
 * the tensor's offsets); the repack is one kernel pair enqueued on hip_stream, allocating nothing.
 * 0: host memory, staged through temporary device buffers and finished before the call returns. */
TURBO_DT_API int turbo_int4_matrix_load(void* matrix, const uint8_t* weight, const uint16_t* scales,
                                        const uint16_t* biases, int weights_on_device, void* hip_stream);
/* Waits for the streams the matrix's loads and products were enqueued on (the whole device when
 * more than four distinct streams were used) and frees it. Calls that use one matrix handle are
 * serialised by the caller. */
TURBO_DT_API void turbo_int4_matrix_destroy(void* matrix);
/* out[i][r] = sum_c (q[r][c] * scale + bias) * x[i][c] for each of `count` (0..32) matrices of one
 * device, in one kernel launch on hip_stream: for example the 8 routed experts' gate and up
 * matrices of a token (16 products of 704 x 2816), then their down matrices. x[i]: [in_dim] FP32,
 * 16-byte aligned; out[i]: [rows] FP32; all device memory. Each out[i] is bit-identical to
 * turbo_int4_matvec on a head of the same matrix. */
TURBO_DT_API int turbo_int4_matvec_grouped(void* const* matrices, int count, const float* const* x,
                                           float* const* out, void* hip_stream);

/*
 * ---- attention of the layer loop -----------------------------------------------------------
 * What stands between the k/q/v projections (turbo_int4_matvec, turbo_int4_matvec_grouped) and the
 * output projection: the norms of the query and key heads with the position rotation, a paged
 * cache that holds keys and values in the tables' own affine format, and attention over it for a
 * batch whose sequences share a prefix. They take the place of the reference's QKVEpilogue and
 * Attention dispatches (shaders/QKVEpilogue.hlsl, shaders/Attention.hlsl).
 *
 * Common rules: head_dim is 64, 128, 256 or 512. Activations are FP32 or BF16 (TURBO_HIDDEN_*),
 * [token][head][head_dim] with the heads of a token contiguous; a stride is the number of elements
 * from one token to the next (0: heads * head_dim), so heads may be slices of a wider row. Buffers
 * are 16-byte aligned and strides a multiple of 16 bytes. The work is enqueued on hip_stream and
 * allocates nothing, so the calls may be captured into a HIP graph. A handle's calls are serialised
 * by the caller; its destroy waits for the streams its calls were enqueued on (the whole device
 * when more than four were used), which must still exist.
 */

/*
 * Keys and values of one layer, quantised as they are written. The cache is `pages` pages of
 * page_tokens tokens; slot s is token s % page_tokens of page s / page_tokens. Every 64 values of a
 * (token, head) are one group: with L = 2^bits - 1, bias = the smallest value rounded down to BF16,
 * scale = (the largest value - bias) / L rounded up to BF16 (at least 2^-126), and a value's code is
 * (value - bias) / scale rounded to the nearest integer, ties to even, limited to 0..L. It reads back
 * as code * scale + bias. A group that holds a value of magnitude 2^103 or more, or NaN, reads back as
 * NaN. The layout in memory is the kernels' own.
 */
typedef struct {
    uint32_t pages;        /* at least 1; pages * page_tokens at most 2^32 - 2 */
    uint32_t page_tokens;  /* 32, 64, 128 or 256 */
    uint32_t kv_heads;     /* 1 .. 1024 */
    uint32_t head_dim;     /* 64, 128, 256 or 512 */
    uint32_t bits;         /* 4 or 8 */
    int device;            /* HIP device ordinal */
} TurboKvCacheDesc;

/* Marks a token that is not written (turbo_kv_cache_write, turbo_qk_norm_rope); like every slot past
 * the cache it reads back as NaN. */
#define TURBO_NO_SLOT 0xFFFFFFFFu

/* 64-token pages, 8 key/value heads of 256 values, 8 bits, no pages yet. */
TURBO_DT_API void turbo_kv_cache_desc_default(TurboKvCacheDesc* out);
/* Allocates the cache: per token and head 2 * (head_dim * bits / 8 + head_dim / 16) bytes. The
 * contents are undefined until they are written. NULL on failure. */
TURBO_DT_API void* turbo_kv_cache_create(const TurboKvCacheDesc* desc);
TURBO_DT_API void turbo_kv_cache_destroy(void* cache);
/* Quantises k and v of `tokens` tokens ([token][kv_heads][head_dim]) into the device slots slots[i].
 * A slot past the cache is skipped. The slots of one call differ: what a repeated one holds afterwards
 * is undefined. */
TURBO_DT_API int turbo_kv_cache_write(void* cache, const void* k, size_t k_stride, const void* v, size_t v_stride,
                                      int dtype, const uint32_t* slots, int tokens, void* hip_stream);
/* Reads `tokens` tokens back (dtype rounds once, to nearest even): out[i] = the token at slots[i], NaN
 * for a slot past the cache. k or v may be NULL. */
TURBO_DT_API int turbo_kv_cache_read(void* cache, const uint32_t* slots, int tokens, int dtype, void* k, size_t k_stride,
                                     void* v, size_t v_stride, void* hip_stream);

enum {
    TURBO_ROPE_HALVES = 0, /* pair i is (x[i], x[i + rotary_dim / 2]); rotary_dim a multiple of 16 */
    TURBO_ROPE_PAIRS = 1   /* pair i is (x[2 i], x[2 i + 1]) */
};
enum { TURBO_NORM_Q = 1u, TURBO_NORM_K = 2u, TURBO_NORM_V = 4u };

/*
 * The norms and the rotation of one layer's heads. A normed head is x / sqrt(mean(x^2) + eps), times
 * the weight where there is one (plain w, as norm_weight of TurboLMHeadDesc; values have none). Then
 * pair i < rotary_dim / 2 of a query or key at position p turns by p * theta^(-2 i / rotary_dim)
 * radians, or p * inv_freq[i] where inv_freq is given (0 leaves a pair as it is); the other elements
 * pass as they are. The angle is within 2^-31 turns of that at every position below 2^32 (a frequency f above 1:
 * f times that).
 */
typedef struct {
    uint32_t head_dim;
    uint32_t rotary_dim;         /* even, 0 .. head_dim */
    int layout;                  /* TURBO_ROPE_* */
    uint32_t norms;              /* TURBO_NORM_* */
    float eps;
    int weights_on_device;       /* of the two norm weights; inv_freq is host memory */
    double theta;
    const double* inv_freq;      /* [rotary_dim / 2], finite, or NULL */
    const uint16_t* q_norm;      /* [head_dim] BF16 or NULL */
    const uint16_t* k_norm;
    int device;
} TurboRotaryDesc;

/* Heads of 256 that rotate whole in halves with theta 10000, queries and keys normed with eps 1e-6,
 * no weights. */
TURBO_DT_API void turbo_rotary_desc_default(TurboRotaryDesc* out);
/* Copies the weights (device weights as the null stream has them) and lays out the frequencies. NULL on failure. */
TURBO_DT_API void* turbo_rotary_create(const TurboRotaryDesc* desc);
TURBO_DT_API void turbo_rotary_destroy(void* rotary);

typedef struct {
    int tokens;                  /* 0 .. 2^28; refused where tokens x heads passes a grid */
    int dtype;                   /* TURBO_HIDDEN_* of q, k, v, q_out and k_out */
    int q_heads;
    int kv_heads;
    const void* q;               /* NULL: no queries */
    const void* k;               /* NULL: no keys */
    const void* v;               /* only for the cache, which needs k and v */
    size_t q_stride, k_stride, v_stride;
    const uint32_t* positions;   /* [tokens] */
    /* where the turned heads go, rounded to dtype once: q (needed with q), k (NULL: only the cache takes
     * them). An output may be its own input, with its stride, and may overlap nothing else. */
    void* q_out;
    void* k_out;
    size_t q_out_stride, k_out_stride;
    /* NULL, or the cache that takes the turned keys and the values, quantised from FP32; token i goes to
     * slots[i] as in turbo_kv_cache_write */
    void* cache;
    const uint32_t* slots;
} TurboQkvInputs;

TURBO_DT_API int turbo_qk_norm_rope(void* rotary, const TurboQkvInputs* in, void* hip_stream);

/*
 * Attention of a batch over the cache. Sequence b holds kv_len[b] tokens: the first prefix_len are the
 * shared prefix, token p of it on page prefix_pages[p / page_tokens], and token prefix_len + j is its
 * own, on page pages[b * page_stride + j / page_tokens]. Its last q_len tokens are the queries, whose
 * own keys are in the cache already: query t is at position kv_len[b] - q_len + t and sees every token
 * up to its own, the last `window` of them where window is not 0.
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * over the tokens that it sees, query head h over key/value head h / (q_heads / kv_heads). A query at
 * a negative position sees nothing and gives zeros (kv_len 0: a padded sequence). A query whose tokens
 * pass its page table, or lie on a page past the cache, gives NaN.
 * The prefix is not read once for each sequence: its products run over the rows of all sequences, 16 or 32 rows of
 * a key/value head at a time (sequences that fill such tiles by themselves take it along with their own
 * tokens). Scores, softmax statistics and sums are FP32; a score beyond FP32's range gives NaN. Keys and
 * values enter as the cache holds them. For FP32 queries, queries and softmax weights keep 22 bits; for BF16
 * ones the weights keep 11; the smallest weighted values 2^-32 of the largest that the row weights. Tokens that
 * a query does not see have no part in its result.
 */
typedef struct {
    int batch;                   /* >= 0 */
    int q_len;                   /* >= 1 */
    int q_heads;                 /* a multiple of the cache's kv_heads */
    int dtype;                   /* TURBO_HIDDEN_* of q and out */
    const void* q;               /* [batch * q_len][q_heads][head_dim] */
    void* out;                   /* the same shape; does not overlap q */
    size_t q_stride, out_stride;
    const uint32_t* kv_len;      /* [batch] */
    uint32_t max_kv_len;         /* what kv_len may reach; sizes the launch, longer sequences are slower, not wrong */
    uint32_t prefix_len;
    const uint32_t* prefix_pages;
    const uint32_t* pages;       /* [batch][page_stride]; NULL when page_stride is 0 */
    uint32_t page_stride;
    uint32_t window;
    float scale;
    /* device scratch of turbo_attention_workspace (turbo_tree_workspace) bytes, 16-byte aligned; calls that may overlap (two
     * streams, two graphs) have one each */
    void* workspace;
    size_t workspace_bytes;
} TurboAttentionInputs;

/* The scratch a call with these sizes needs (0: none); pointers are not looked at. With a q_len of at most 64 it serves
 * turbo_tree_attention too, which has use for more (turbo_tree_workspace). */
TURBO_DT_API int turbo_attention_workspace(void* cache, const TurboAttentionInputs* in, size_t* bytes);
TURBO_DT_API int turbo_prefix_attention(void* cache, const TurboAttentionInputs* in, void* hip_stream);

/*
 * Attention of drafted trees: turbo_prefix_attention for sequences whose last q_len tokens (1 .. 64) are a tree's
 * nodes in place of a run. masks: [batch][q_len] device words, bit j of one: the query sees node j of its own
 * sequence (turbo_batch_plan makes them of the nodes' parents; bits from q_len on are ignored). A query sees the
 * kv_len[b] - q_len tokens before the tree and the nodes of its mask, in this order the last `window` of them
 * where window is not 0. A mask of 0 marks an absent node, which gives zeros; nodes that a query does not see
 * have no part in its result, whatever their slots hold. Everything else is as there, but that
 * for BF16 queries of many rows the keys and values before the tree may be rounded to fp16, 2^-11 of each and 2^-18 of
 * the largest of its head, and the smallest weighted values to 2^-20 of the largest.
 */
TURBO_DT_API int turbo_tree_attention(void* cache, const TurboAttentionInputs* in, const uint64_t* masks, void* hip_stream);
/* The scratch with which a tree's call of these sizes is fastest (of many rows 512 MB of partial results at most). The call
 * takes less, down to this or what turbo_attention_workspace gives, whichever is smaller, and then splits the keys into
 * fewer parts: how much there is decides the last bits of the results. */
TURBO_DT_API int turbo_tree_workspace(void* cache, const TurboAttentionInputs* in, size_t* bytes);

/*
 * Moves tokens inside the cache, codes, scales and biases bit by bit: the token at source[r * width + i] goes to
 * target[r * width + i] for `rows` rows of `width` (1 .. 64) moves, device slots. What a row moves is read before
 * the row writes anything, so a row may write slots that it reads; the targets of a row differ, and different
 * rows share no slot that one of them writes. A move from or to a slot past the cache (TURBO_NO_SLOT) is skipped.
 */
TURBO_DT_API int turbo_kv_cache_move(void* cache, const uint32_t* source, const uint32_t* target, int rows, int width,
                                     void* hip_stream);

/*
 * ---- a serving step's requests --------------------------------------------------------------
 * What the calls above take as slots, positions, lengths, page tables and masks, made on the device from the
 * lengths of the sequences, and attention over prompts that are not in a cache yet. No counterpart in the reference
 * (one sequence, a ring of 4096). The calls have no handle: they run on the device that they name, on hip_stream,
 * allocate nothing and may be captured into a HIP graph. The arrays of a call that it writes share no bytes with each other or
 * with those that it reads, where nothing else is said.
 */

/* A page that a sequence needs and the pool did not have. */
#define TURBO_NO_PAGE 0xFFFFFFFFu

/*
 * One step of a batch: sequence b holds past_len[b] tokens and adds new_len[b]. The first prefix_len tokens of every
 * sequence are the shared prefix, on pages of its own; the others are on the sequence's pages, as
 * TurboAttentionInputs has them. The table of sequence b holds held[b] pages. It gets those that it lacks from the
 * end of the pool's list, in the order of the sequences and of their pages: the k-th page taken is
 * free_pages[free_count - 1 - k]. Where the pool is empty the table gets TURBO_NO_PAGE, held_out does not count it,
 * and the tokens on it get TURBO_NO_SLOT, as do tokens past the table (totals[3] counts such pages; once the pool has
 * pages again the same plan gets them).
 *
 * The tokens added are packed, sequence after sequence (row_tokens 0), or lie in rows of row_tokens, of which a
 * sequence fills the first new_len (what passes row_tokens is left out). Entries that no token has get position 0 and
 * TURBO_NO_SLOT. With parents the rows are drafted trees: node t of sequence b hangs on node parents[b][t] < t, or on
 * the sequence's last token (-1). A node with any other parent, past new_len, or whose parent is absent is absent.
 * Its mask holds the bits of its ancestors and its own; its position is past_len plus the number of its ancestors; its
 * slot is that of token past_len + t.
 */
typedef struct {
    int batch;                      /* 0 .. 8192 */
    uint32_t page_tokens;           /* the caches' */
    uint32_t prefix_len;
    const uint32_t* past_len;       /* [batch], the prefix included */
    const uint32_t* new_len;        /* [batch] */
    uint32_t row_tokens;
    uint32_t max_tokens;            /* entries of positions and slots, at most 2^28; batch * row_tokens for rows */
    const int32_t* parents;         /* [batch][row_tokens] or NULL; row_tokens is at most 64 then */
    uint32_t* pages;                /* [batch][page_stride], the new pages are written */
    uint32_t page_stride;
    const uint32_t* held;           /* [batch] */
    const uint32_t* free_pages;     /* [free_capacity] */
    const uint32_t* free_count;     /* [1] */
    uint32_t free_capacity;
    /* the pool's state after the step; may be held and free_count themselves */
    uint32_t* held_out;
    uint32_t* free_count_out;
    /* results, each may be NULL */
    uint32_t* starts;               /* [batch + 1] first entry of every sequence */
    uint32_t* kv_len;               /* [batch] past + new; for rows past + row_tokens, as the attention counts its
                                       queries (0 for a sequence that adds nothing); may be past_len itself */
    uint32_t* positions;            /* [max_tokens] */
    uint32_t* slots;                /* [max_tokens] */
    uint64_t* masks;                /* [batch][row_tokens], with parents */
    uint32_t* totals;               /* [4] tokens added, tokens left out, pages taken, pages missing */
    int device;                     /* HIP device ordinal */
} TurboBatchPlan;
TURBO_DT_API int turbo_batch_plan(const TurboBatchPlan* in, void* hip_stream);

/* Gives pages back: sequence b keeps those of its first keep_len[b] tokens (the prefix included; 0: none), the others
 * go to the end of the pool's list in the order of the sequences. The list has room for every page of the caches. */
typedef struct {
    int batch;                      /* 0 .. 8192 */
    uint32_t page_tokens;
    uint32_t prefix_len;
    const uint32_t* keep_len;       /* [batch] */
    const uint32_t* pages;          /* [batch][page_stride] */
    uint32_t page_stride;
    uint32_t* held;                 /* [batch], updated */
    uint32_t* free_pages;           /* [free_capacity], updated */
    uint32_t* free_count;           /* [1], updated */
    uint32_t free_capacity;
    int device;
} TurboPagesRelease;
TURBO_DT_API int turbo_pages_release(const TurboPagesRelease* in, void* hip_stream);

/*
 * The path of every tree that the model confirms. Node 0 is the token that the step before drew, so it is kept;
 * then, from the last kept node on, the first child whose token is the one chosen after that node (turbo_lmhead_step's
 * tokens over the nodes as rows; 0xFFFFFFFF, its mark of a degenerate row, confirms nothing). next is the choice after the last kept node:
 * node 0 of the following step. The i-th kept node's key and value belong at the slot of node i: source and target
 * say so to turbo_kv_cache_move, once for each layer's cache. Parents as in TurboBatchPlan. A result may be an input itself, of
 * the same size (length past_len, for one).
 */
typedef struct {
    int batch;                      /* 0 .. 2^20 */
    uint32_t row_tokens;            /* 1 .. 64 */
    const int32_t* parents;         /* [batch][row_tokens] */
    const uint32_t* new_len;        /* [batch] nodes of each tree */
    const uint32_t* tokens;         /* [batch][row_tokens] */
    const uint32_t* chosen;         /* [batch][row_tokens] */
    const uint32_t* past_len;       /* [batch], for length */
    const uint32_t* slots;          /* [batch][row_tokens], for source and target */
    uint32_t* kept;                 /* [batch] nodes kept */
    uint32_t* next;                 /* [batch]; 0xFFFFFFFF where nothing is kept */
    /* each may be NULL, source and target together */
    uint32_t* length;               /* [batch] past_len + kept */
    uint32_t* path;                 /* [batch][row_tokens] the kept nodes, then 0xFFFFFFFF */
    uint32_t* source;               /* [batch][row_tokens] their slots, then TURBO_NO_SLOT */
    uint32_t* target;               /* [batch][row_tokens] where they belong, then TURBO_NO_SLOT */
    int device;
} TurboTreeAccept;
TURBO_DT_API int turbo_tree_accept(const TurboTreeAccept* in, void* hip_stream);

/*
 * Causal attention of whole prompts over their own keys and values, before or without a cache. Sequence b is rows
 * starts[b] .. starts[b + 1] - 1 of q, k, v and out (starts is not decreasing; rows past `tokens` are left out).
 * Query i of it sees keys 0 .. i, the last `window` of them where window is not 0:
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * query head h over key/value head h / (q_heads / kv_heads). Buffers as the layer loop's common rules have them, with
 * strides of at most 2^24 elements. Rows of no sequence are left as they were. Products q . k, scores, softmax statistics and
 * sums are FP32. BF16 inputs are multiplied as they are, their softmax weights rounded to BF16 (2^-8 of each at most). FP32
 * ones are multiplied in FP32 or, for calls of many rows and all with heads of 512, in 16-bit parts: of queries and keys 2^-22 of
 * each number and 2^-39 of the largest of its head may be lost then, of weights and values 2^-24.
 * NaN in a query or in a key that it sees gives NaN, as do an infinity in a query and a product or score of +infinity; a key whose
 * score is -infinity has a weight of 0 (where no other is left, NaN). NaN or an infinity in a value that it sees gives the same or
 * NaN in its column. What a query does not see has no part in its result. `tokens`, the rows that the buffers have, sizes the launch.
 */
typedef struct {
    int batch;                   /* 0 .. 2^20 */
    int tokens;                  /* rows of the buffers, 0 .. 2^28 */
    int q_heads;                 /* a multiple of kv_heads */
    int kv_heads;
    uint32_t head_dim;           /* 64, 128, 256 or 512 */
    int dtype;                   /* TURBO_HIDDEN_* of q, k, v and out */
    const void* q;               /* [tokens][q_heads][head_dim] */
    const void* k;               /* [tokens][kv_heads][head_dim] */
    const void* v;
    void* out;                   /* as q; overlaps nothing else */
    size_t q_stride, k_stride, v_stride, out_stride;
    const uint32_t* starts;      /* [batch + 1] */
    uint32_t window;
    float scale;                 /* magnitude below 2^127 */
    int device;                  /* HIP device ordinal */
} TurboPromptInputs;
TURBO_DT_API int turbo_prompt_attention(const TurboPromptInputs* in, void* hip_stream);

/*
 * Embedding lookup on the same tied table (shaders/EmbedLookup.hlsl:1-45; CPU
 * src/cpu_reference.cpp:108-124 and :323-329): out[i] = row tokens[i] dequantised as
 * (float)q * scale + bias, times sqrtf(hidden). tokens: [n] device ids, out: [n][hidden] FP32
 * device, stream-ordered on the handle's stream. The reference throws for an id past the
 * vocabulary (:325-327); here, where ids stay on the device, such a row is written as NaN.
 */
TURBO_DT_API int turbo_lmhead_embed(void* handle, const uint32_t* tokens, int n, float* out);

/* ---- kernel-level entry points (one per reference kernel on the path) -------------------- */

/* RMSNormK with model.norm.weight (shaders/RMSNormK.hlsl:25-61; src/cpu_reference.cpp:43-52).
 * x, out: [batch][hidden] FP32. */
TURBO_DT_API int turbo_lmhead_rms_norm(void* handle, const float* x, int batch, float* out);

/* GemvInt4 over the tied table (shaders/GemvInt4.hlsl:18-38, src/runner.cpp:429-442, :773),
 * followed by Softcap when apply_softcap (shaders/Softcap.hlsl:18-30, src/runner.cpp:774-779).
 * x: [batch][hidden] (TURBO_HIDDEN_*, already normalised), logits: [batch][vocab] FP32. */
TURBO_DT_API int turbo_lmhead_logits(void* handle, const void* x, int x_dtype, int batch,
                                     int apply_softcap, float* logits);

/* LMHeadGreedy + ArgmaxReduce (shaders/LMHeadGreedy.hlsl:28-73, ArgmaxReduce.hlsl:21-62):
 * argmax of the softcapped logits, ties to the lowest row. tokens: [batch]. */
TURBO_DT_API int turbo_lmhead_greedy(void* handle, const void* x, int x_dtype, int batch,
                                     uint32_t* tokens);

/* Softcap in place on n floats (shaders/Softcap.hlsl:18-30). stream may be NULL. */
TURBO_DT_API int turbo_softcap(void* hip_stream, float* z, size_t n, float cap);

/* apply_repetition_penalty in place on one row (src/sampling.cpp:74-90). stream may be NULL. */
TURBO_DT_API int turbo_apply_repetition_penalty(void* hip_stream, float* logits, uint32_t vocab,
                                                const uint32_t* history, uint32_t n,
                                                float penalty, float softcap);

/*
 * Sampling on caller-provided logits (sample_token, src/sampling.cpp:92-169, plus the
 * modifiers of turbo_lmhead_step). logits: [batch][vocab], modified in place by the
 * modifiers. in->hidden and in->hidden_dtype are ignored. out->logits is ignored.
 */
TURBO_DT_API int turbo_sample_logits(void* handle, float* logits, const TurboStepInputs* in,
                                     const TurboStepOutputs* out);

/* ---- sampling without a handle or an allocation ---------------------------------------- */

#define TURBO_NOALLOC_MAX_BATCH 4
#define TURBO_NOALLOC_MAX_VOCAB 262144

/*
 * turbo_sample_logits without a handle and without allocating: the modifiers of
 * TurboStepInputs and the sampler (sample_token semantics, src/sampling.cpp:92-169) over
 * caller logits [batch][vocab], modified in place, tokens (and reports) into `out`. No
 * counterpart in the reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). It calls no hipMalloc,
 * hipFree or allocating routine; its working memory is one static device array of about 14 MiB
 * per GPU (held until the process ends), sized for batch <= TURBO_NOALLOC_MAX_BATCH and
 * vocab <= TURBO_NOALLOC_MAX_VOCAB, with at most 8192 logit-bias entries per row. Larger inputs
 * fail with a clear error. The work is enqueued on hip_stream (NULL = the null stream) of the
 * current device; the first call on a device clears the array on that stream. Every call on a GPU
 * shares that GPU's array: calls that overlap on one GPU race, so the caller serialises them.
 * in->hidden and out->logits are ignored; TURBO_STATUS_HISTORY_FULL is reported per row only.
 */
TURBO_DT_API int turbo_sample_logits_noalloc(void* hip_stream, uint32_t vocab, float final_logit_softcap,
                                             float* logits, const TurboStepInputs* in,
                                             const TurboStepOutputs* out);

/* ---- measurement ------------------------------------------------------------------------- */

/* When enabled, the head kernel (the int4 GEMV / MFMA kernel) is launched with HIP start and
 * stop events on the handle's stream. enable = 1 times every launch; enable = N > 1 times every
 * N-th launch (the events add a few microseconds of gap around the timed launch, so sampling
 * keeps a loop's throughput representative). turbo_lmhead_head_kernel_time synchronises and
 * returns the summed milliseconds and the number of timed launches since the last reset. */
TURBO_DT_API int turbo_lmhead_enable_head_timing(void* handle, int enable);
TURBO_DT_API int turbo_lmhead_head_kernel_time(void* handle, double* total_ms, int* launches,
                                               int reset);

#ifdef __cplusplus
}
#endif

#endif /* TURBO_DECODE_TAIL_H */
