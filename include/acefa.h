/*
 * acefa.h -- C ABI of the B200 (sm_100a) attention engine behind acestep.cpp's
 * ggml_flash_attn_ext operator.
 *
 * The engine replaces the CUDA-side execution of one GGML_OP_FLASH_ATTN_EXT
 * graph node.  acestep.cpp creates those nodes at
 *   src/qwen3-lm.h:465-469    (LM prefill / single decode, PREC_F32)
 *   src/qwen3-lm.h:789-794    (LM batched CFG decode, PREC_F32)
 *   src/qwen3-enc.h:195-199   (text / lyric / timbre / FSQ encoders)
 *   src/dit-graph.h:227-231   (DiT self-attention)
 *   src/dit-graph.h:348-352   (DiT cross-attention)
 * and ggml's CUDA backend executes them in its per-node switch
 * (case GGML_OP_FLASH_ATTN_EXT -> ggml_cuda_flash_attn_ext(ctx, dst) in the
 * ggml fork that acestep.cpp pins as a submodule, .gitmodules:1-3).  That call
 * is what acefa_flash_attn_ext() replaces; acefa_supports() replaces the
 * GGML_OP_FLASH_ATTN_EXT branch of ggml_backend_cuda_device_supports_op, which
 * acestep.cpp's static_graph_alloc consults (src/static-graph.h:12-19).
 *
 * Tensors use ggml's conventions: ne[0] innermost, nb[] byte strides, type ids
 * equal to enum ggml_type.  All data pointers are device pointers owned by the
 * caller (ggml's allocator).  No entry point allocates device memory or aborts;
 * acefa_flash_attn_ext() also never synchronises, so it is safe inside
 * CUDA-graph stream capture.
 */
#ifndef ACEFA_H
#define ACEFA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define ACEFA_API __attribute__((visibility("default")))
#else
#define ACEFA_API
#endif

/* Same numeric values as enum ggml_type. */
typedef enum acefa_type {
    ACEFA_TYPE_F32  = 0,
    ACEFA_TYPE_F16  = 1,
    ACEFA_TYPE_Q8_0 = 8,
    ACEFA_TYPE_I8   = 24,
    ACEFA_TYPE_I32  = 26,
    ACEFA_TYPE_BF16 = 30,
} acefa_type;

/* Same numeric values as enum ggml_prec (ggml_flash_attn_ext_set_prec). */
typedef enum acefa_prec {
    ACEFA_PREC_DEFAULT = 0,
    ACEFA_PREC_F32     = 10,
} acefa_prec;

typedef enum acefa_status {
    ACEFA_OK             = 0,
    ACEFA_ERR_NULL       = -1, /* a required tensor or pointer is NULL */
    ACEFA_ERR_TYPE       = -2, /* unsupported element type */
    ACEFA_ERR_SHAPE      = -3, /* shapes violate the ggml_flash_attn_ext contract */
    ACEFA_ERR_LAYOUT     = -4, /* stride/alignment this engine does not support */
    ACEFA_ERR_WORKSPACE  = -5, /* workspace too small or not 256-B aligned */
    ACEFA_ERR_CUDA       = -6, /* a CUDA runtime/driver call failed */
    ACEFA_ERR_DEVICE     = -7, /* current device is not sm_100 */
    ACEFA_ERR_DEVICE_TIMEOUT = -8, /* a bounded device-side wait expired */
    ACEFA_ERR_NOALLOC_LIMIT  = -9, /* operands need more scratch than acefa_flash_attn_ext_noalloc's fixed buffer */
} acefa_status;

/* ggml_tensor reduced to what the operator reads. */
typedef struct acefa_tensor {
    int32_t type;  /* acefa_type */
    int64_t ne[4]; /* elements per dimension, ne[0] innermost */
    size_t  nb[4]; /* byte strides; for Q8_0 nb[0] = 34 (block bytes) */
    void   *data;  /* device pointer */
} acefa_tensor;

/*
 * dst = softmax(scale * Q K^T [softcap] + slope * mask [+ sinks]) V, permuted.
 *
 *   q     [D,  n_q,  Hq,  B ]  F32, any strides with nb[0] == 4
 *   k     [D,  n_kv, Hkv, Bk]  F16, BF16 or Q8_0; Hq % Hkv == 0, B % Bk == 0
 *   v     [Dv, n_kv, Hkv, Bk]  same type as k, Dv == D
 *   mask  [>=n_kv, >=n_q, Hm, Bm] F16 or NULL; Hq % Hm == 0, B % Bm == 0
 *   sinks [Hq] F32 or NULL (extra softmax logit per head, no value row)
 *   dst   [Dv, Hq, n_q, B] F32
 *
 * scale, max_bias (ALiBi) and logit_softcap have ggml's meaning.  prec is
 * accepted for either value; accumulation is always F32.  stream is a
 * cudaStream_t (NULL = legacy default stream); a kernel directly ahead on it
 * that lets its dependents start early (programmatic launch) writes q, masks and
 * positions before it does so.  workspace must hold
 * acefa_workspace_bytes() bytes, 256-B aligned, caller-owned; its contents need
 * no initialisation and are dead after the call's kernels finish.
 * Returns ACEFA_OK or a negative acefa_status; launches nothing on error.
 */
ACEFA_API int acefa_flash_attn_ext(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                   const acefa_tensor *mask, const acefa_tensor *sinks, const acefa_tensor *dst,
                                   float scale, float max_bias, float logit_softcap, int prec, void *stream,
                                   void *workspace, size_t workspace_bytes);

/*
 * The same operator for callers that cannot hand the engine any device memory:
 * hosts whose device memory is entirely owned by another allocator (a ggml
 * backend whose graph allocator has planned every buffer, a plugin inside a
 * framework that forbids foreign allocations), threads that must never block
 * (cudaMalloc can synchronise the whole device), and builds that forbid runtime
 * allocation after start-up.  No counterpart in the reference: ggml's CUDA
 * backend always draws flash-attention scratch from its own memory pool.
 *
 * Arguments and results are those of acefa_flash_attn_ext() without the
 * workspace pair.  The scratch is a fixed 8 MiB array inside the library, one
 * per GPU, held from library load until process exit; only the dense
 * (query-heavy) path uses it -- its mask-class table, the partial results of
 * its last-wave key-range split, F16 copies of BF16 K/V when they fit -- while
 * decode nodes need none.  The call plans its work for that 8 MiB (the dense
 * path shrinks or drops its split and skips the BF16 copies to fit, exactly as
 * acefa_flash_attn_ext would with an 8 MiB workspace); operands that need more
 * even then -- a mask-class table over 8 MiB -- are refused with
 * ACEFA_ERR_NOALLOC_LIMIT and nothing is launched.  The first call on each
 * device looks up that array's device address (with the device current), so
 * make that first call before any stream capture.  The address is kept for the
 * life of the process: after cudaDeviceReset() on a device this entry (like the
 * engine's device error word) must not be used on it again.  Every call on a device
 * shares the array: calls whose kernels may overlap on the GPU (other streams or
 * other threads without ordering) race and must be serialised by the caller.
 * Nothing is allocated, freed or zeroed by the call.
 */
ACEFA_API int acefa_flash_attn_ext_noalloc(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                           const acefa_tensor *mask, const acefa_tensor *sinks,
                                           const acefa_tensor *dst, float scale, float max_bias, float logit_softcap,
                                           int prec, void *stream);

/*
 * Multi-GPU extension; no counterpart in the reference, which runs every module
 * on one device.  The operator with its result also written to up to
 * ACEFA_MAX_MIRRORS further buffers ("mirrors"), each laid out exactly like dst
 * (same ne and nb) at another address: typically this rank's head slice of a
 * peer GPU's full output, mapped with acefa_peer_import().  The kernels' output
 * stage stores every row to dst and to each mirror (plain stores, over NVLink
 * for peer memory), so a head-sharded attention layer assembles its full
 * output on every GPU with no separate all-gather.  Each mirror must be
 * congruent to dst modulo 16 bytes.  n_mirrors == 0 is acefa_flash_attn_ext().
 * The call signals nothing to the peers: before a peer reads its output the
 * caller orders it after this stream's work (a collective on this stream after
 * the call, or an IPC event).  Returns ACEFA_ERR_NULL / ACEFA_ERR_LAYOUT for a
 * NULL or misaligned mirror, ACEFA_ERR_SHAPE for n_mirrors out of range.
 */
#define ACEFA_MAX_MIRRORS 7
ACEFA_API int acefa_flash_attn_ext_mirrored(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                            const acefa_tensor *mask, const acefa_tensor *sinks,
                                            const acefa_tensor *dst, float scale, float max_bias,
                                            float logit_softcap, int prec, void *const *mirrors, int n_mirrors,
                                            void *stream, void *workspace, size_t workspace_bytes);

/*
 * The operator fused with the KV-cache append that precedes it in a decode
 * step.  The reference writes the new row with two ggml_set_rows nodes (K and V
 * at src/qwen3-lm.h:776-777, inside qw3lm_forward_batch) and then runs the
 * attention node over the cache views; this entry does both in one launch.
 *
 *   k_new, v_new  [D, 1, Hkv, Bk] F32, nb[0] == 4: the new row of every
 *                 (kv head, set), already projected, normed and rotated
 *   pos           device array of Bk int64: the cache row (0 <= pos < n_kv of
 *                 the k/v views) that receives set s's new row
 *
 * Row pos[s] of every head of set s in k and v is overwritten with k_new /
 * v_new converted to the cache type (F16 / BF16 rounded to nearest even; Q8_0
 * by ggml's reference quantiser: d = amax/127, q = roundf(x * (1/d)), d as f16), and
 * the attention then reads the updated cache exactly as acefa_flash_attn_ext
 * would have after the two set_rows.  The k and v views must be writable and
 * each (head, set) row written once: sets whose views alias each other, or a
 * mask that hides row pos[s], are the caller's concern.  Served by the decode
 * path only (query rows per kv head <= 64, i.e. decode steps); other shapes
 * return ACEFA_ERR_SHAPE.  A pos outside [0, n_kv) leaves that set's row
 * unwritten and raises device error 5 (acefa_device_error()).  Other
 * arguments and results are those of acefa_flash_attn_ext().
 */
ACEFA_API int acefa_flash_attn_ext_append(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                          const acefa_tensor *mask, const acefa_tensor *sinks,
                                          const acefa_tensor *dst, float scale, float max_bias, float logit_softcap,
                                          int prec, const acefa_tensor *k_new, const acefa_tensor *v_new,
                                          const int64_t *pos, void *stream, void *workspace, size_t workspace_bytes);

/*
 * A mask given by its rule instead of an f16 tensor.  acestep.cpp fills these
 * masks on the host and the attention node reads them back from HBM: the LM
 * prefill causal mask (src/qwen3-lm.h:597-609), the batched decode validity
 * mask (src/qwen3-lm.h:872-881), the DiT sliding window sa_mask_sw and the
 * cross-attention padding ca_mask (src/dit-sampler.h:262-311).
 * Key j is visible to query i (0-based within n_q) of batch b when
 *   ACEFA_MASK_CAUSAL   j <= pos0[b] + i   (LM prefill with the cache holding
 *                       pos0 earlier tokens; a decode step is i = 0, keys
 *                       0 .. kv_pos)
 *   ACEFA_MASK_WINDOW   |i - j| <= window  (DiT self-attention, sliding-window
 *                       layers; where the reference's window is off -- win <= 0
 *                       or S <= win -- the node is unmasked: pass no mask)
 *   ACEFA_MASK_PADDING  j < len[b]         (DiT cross-attention padding)
 * Visible keys add 0 and hidden keys -inf, exactly as the equivalent f16
 * mask would; results are bit-identical to acefa_flash_attn_ext with that mask.
 * pos0 / len are read for b < B (at most ACEFA_MASK_GEN_MAX_BATCH batches).
 */
#define ACEFA_MASK_GEN_MAX_BATCH 32
typedef enum acefa_mask_kind {
    ACEFA_MASK_CAUSAL  = 1,
    ACEFA_MASK_WINDOW  = 2,
    ACEFA_MASK_PADDING = 3,
} acefa_mask_kind;

typedef struct acefa_mask_gen {
    int32_t kind;    /* acefa_mask_kind */
    int32_t window;  /* ACEFA_MASK_WINDOW */
    int64_t pos0[ACEFA_MASK_GEN_MAX_BATCH];  /* ACEFA_MASK_CAUSAL */
    int64_t len[ACEFA_MASK_GEN_MAX_BATCH];   /* ACEFA_MASK_PADDING */
} acefa_mask_gen;

/* acefa_flash_attn_ext() with the mask given by rule (mask_gen, host memory,
 * read during the call) instead of a tensor: no mask is read on the device and
 * the dense path needs no mask-classification pass.  The rule is copied into
 * the launch, so mask_gen may be reused or freed once the call returns.
 * acefa_workspace_bytes(q, k, v, NULL, dst) is enough workspace.  Returns
 * ACEFA_ERR_SHAPE for an unknown kind, B > ACEFA_MASK_GEN_MAX_BATCH with a
 * per-batch kind (CAUSAL, PADDING), or a negative window. */
ACEFA_API int acefa_flash_attn_ext_gen(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                       const acefa_mask_gen *mask_gen, const acefa_tensor *sinks,
                                       const acefa_tensor *dst, float scale, float max_bias, float logit_softcap,
                                       int prec, void *stream, void *workspace, size_t workspace_bytes);

/*
 * The attention prologue acestep.cpp runs as separate graph nodes before the
 * attention node (src/qwen3-lm.h:423-431, src/dit-graph.h:181-197):
 *   y = ggml_rms_norm(x, eps) * norm_weight        (per row of D values)
 *   y = ggml_rope_ext(y, positions, mode 2 = NEOX, n_dims = D, freq_base =
 *       theta_base, freq_scale 1, no YaRN)
 * i.e. pair k < D/2 rotates (y[k], y[k + D/2]) by positions[..] *
 * theta_base^(-2k/D).  Row i of batch b has position positions[i + b * n],
 * n being the rows per batch of the tensor it applies to (n_q for Q; for a
 * decode step's new K row, n = 1: positions[set]).
 */
typedef struct acefa_rope_norm {
    const float   *norm_weight;  /* [D] f32, device; NULL = no RMSNorm */
    float          eps;          /* rms_norm_eps */
    float          theta_base;   /* rope_theta; 0 = no RoPE */
    const int32_t *positions;    /* int32, device (ggml's positions tensor); unused without RoPE */
} acefa_rope_norm;

/*
 * Options of acefa_flash_attn_ext_fused().  Zero-initialise and set what is
 * used; every member may be NULL / 0.
 */
typedef struct acefa_op_ext {
    const acefa_mask_gen  *mask_gen;    /* mask by rule; `mask` must then be NULL */
    const acefa_rope_norm *q_prologue;  /* applied to each Q row as the kernels load it */
    /* Fused KV-cache append (decode path), as acefa_flash_attn_ext_append: */
    const acefa_tensor    *k_new, *v_new;
    const int64_t         *append_pos;
    const acefa_rope_norm *k_prologue;  /* applied to k_new before it is converted and stored */
    /* Mirrors, as acefa_flash_attn_ext_mirrored: */
    void *const           *mirrors;
    int                    n_mirrors;
} acefa_op_ext;

/* The operator with any combination of the fusions above (NULL ext = plain
 * acefa_flash_attn_ext).  Q given with a q_prologue is the raw projection
 * output (before RMSNorm and RoPE), in the same [D, n_q, Hq, B] view. */
ACEFA_API int acefa_flash_attn_ext_fused(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                         const acefa_tensor *mask, const acefa_tensor *sinks,
                                         const acefa_tensor *dst, float scale, float max_bias,
                                         float logit_softcap, int prec, const acefa_op_ext *ext, void *stream,
                                         void *workspace, size_t workspace_bytes);

/*
 * K / V preparation for the dense path in one pass: k_dst = RoPE(RMSNorm(k_src))
 * and v_dst = v_src, converted to the destination type (F16 or BF16), at any
 * strides on either side (so the permute of the reference's graph and a
 * write into a KV-cache window are both just destination views).  Replaces
 * the rms_norm, mul, rope, cont and cast / set_rows nodes of
 * src/dit-graph.h:181-213 and src/qwen3-lm.h:423-449.  k_src / v_src: F32
 * [D, rows, H, B] with rows * H * B < 2^31; k_dst / v_dst: the same ne.
 * v_src / v_dst may be NULL.  Positions index as positions[row + b * rows].
 */
ACEFA_API int acefa_kv_prologue(const acefa_tensor *k_src, const acefa_tensor *v_src, const acefa_tensor *k_dst,
                                const acefa_tensor *v_dst, const acefa_rope_norm *k_prologue, void *stream);

/*
 * CUDA IPC through the ABI, so a host without CUDA bindings can map peer
 * buffers.  acefa_peer_export: an opaque handle (ACEFA_PEER_HANDLE_BYTES bytes)
 * for the allocation holding ptr, plus ptr's byte offset inside it.
 * acefa_peer_import (another process of the same node, its own device current):
 * maps that allocation with peer access enabled and returns the address that
 * corresponds to the exported ptr.  acefa_peer_release: unmaps an address
 * acefa_peer_import returned.  All three return ACEFA_OK or ACEFA_ERR_CUDA /
 * ACEFA_ERR_NULL.
 */
#define ACEFA_PEER_HANDLE_BYTES 64
ACEFA_API int acefa_peer_export(const void *ptr, void *handle, uint64_t *offset);
ACEFA_API int acefa_peer_import(const void *handle, uint64_t offset, void **ptr);
ACEFA_API int acefa_peer_release(void *ptr);

/*
 * CFG combine + logit compaction of a batched LM decode step on the device:
 * the host loop of src/pipeline-lm.cpp:471-492 (and, with eos_idx < 0 and the
 * range [0, V), the full-vocabulary combines of :104-108, :193-199, :364-370),
 * so that only the compact rows cross to the host.  cond / uncond: F32 logits,
 * sequence a's rows at cond + a * row_stride and uncond + a * row_stride (in
 * the reference's batch layout uncond = cond + n * row_stride); uncond NULL:
 * no CFG (the reference's use_cfg false), a plain gather.  compact: n rows of
 * cols = code_count + (eos_idx >= 0) floats, contiguous:
 *   column 0            <- logit eos_idx            (only when eos_idx >= 0)
 *   following columns   <- logits code_offset .. code_offset + code_count - 1
 * each u + cfg_scale * (c - u) with every operation rounded to F32 on its own
 * (no FMA), bit-identical to the reference's x86-64 host arithmetic.
 * compact must not overlap cond or uncond, except compact == cond with
 * eos_idx < 0, code_offset 0 and code_count == row_stride (the in-place
 * full-row combine).  n <= 65535.  Stream-ordered, one launch (none for
 * n == 0, which accepts NULL buffers).  Returns ACEFA_ERR_NULL, ACEFA_ERR_SHAPE (a column outside the row,
 * n out of range), ACEFA_ERR_LAYOUT (misaligned or overlapping buffers).
 */
ACEFA_API int acefa_cfg_logit_combine(const float *cond, const float *uncond, int64_t row_stride, int n,
                                      int eos_idx, int code_offset, int code_count, float cfg_scale,
                                      float *compact, void *stream);

/* ------------------------------------------------------------------------
 * A KV cache held in 8 bits with one scale per block of 64 tokens and head.
 * No counterpart in the reference, whose cache is F16 (src/qwen3-lm.h:228-229);
 * it takes the place of one layer's F16 K and V ([D, n_max, Hkv, n_sets]) at
 * a little over half the bytes.  Row j of (head h, set s) stands for the values
 *   k[d, j, h, s] * k_scale[j / 64, h, s]         (each product rounded to F32)
 * and likewise for v.  k, v: I8 [D, n_max, Hkv, Bk], D 64 or 128, nb[0] == 1,
 * data and nb[1..3] multiples of 16 bytes, not 0; k_scale, v_scale: F32
 * [ceil(n_max / 64), Hkv, Bk], nb[0] == 4.  A value is off by at most half its
 * block's scale when it is stored, and by half the new scale whenever that
 * grows: coarser than Q8_0 with its scale per 32 values (a root mean square of 0.9 %
 * of normal rows stored at once and 1.2 % one by one, Q8_0 0.5 %).  1 <= Bk <= ACEFA_KV8_MAX_SETS,
 * Hkv <= 4096.  A cache needs no initialisation: rows at or past a set's
 * length are never read as values.
 *
 * Every array of lengths, positions or offsets below is device memory that the
 * kernels read, so a captured CUDA graph replays with new lengths.  The
 * entries launch on `stream` only, allocate nothing and never synchronise.
 */
#define ACEFA_KV8_BLOCK    64
#define ACEFA_KV8_MAX_SETS 1024
typedef struct acefa_kv8_cache {
    acefa_tensor k, v;             /* I8  [D, n_max, Hkv, Bk] */
    acefa_tensor k_scale, v_scale; /* F32 [ceil(n_max / 64), Hkv, Bk] */
} acefa_kv8_cache;

/*
 * Stores new rows: a decode step's one row per set, or whole prompts.
 *   k_new, v_new  [D, rows, Hkv, 1], both F32, F16 or BF16, nb[0] = the element
 *                 size: the sets' new rows behind one another
 *   cu_rows       int32 [Bk + 1], device: set s's rows are cu_rows[s] ..
 *                 cu_rows[s + 1] - 1; NULL: rows / Bk rows for every set
 *   pos           int32 [Bk], device: the cache row of set s's first new row;
 *                 its length becomes pos[s] + its number of new rows
 * A block's scale is d = amax / 127 (F32 division) of its new rows, and where
 * rows before pos[s] stay in the block not below the scale they have.  New
 * values become x / d rounded to the nearest integer, ties to even (0 where
 * d is 0); where d grew, the rows that stay are rounded again: q * d_old / d.
 * Both quotients are rounded once, exactly.  A NaN or an infinity among the
 * new rows makes their block's scale NaN, which it stays while a row of the
 * block stays.  Rows of the last block behind the
 * new length are left as they are.  A set whose rows are no rows of the
 * cache or of k_new (a negative pos, an end past n_max, offsets that
 * decrease or leave [0, rows]) is left unwritten and raises device error 5
 * (acefa_device_error()); where offsets decrease, other sets may be left
 * unfinished.  k_new and v_new must not overlap the cache.
 */
ACEFA_API int acefa_kv8_store(const acefa_kv8_cache *cache, const acefa_tensor *k_new, const acefa_tensor *v_new,
                              const int32_t *cu_rows, const int32_t *pos, void *stream);

/*
 * Reads the cache back as values: k_dst, v_dst [D, n, Hkv, Bk], n <= n_max,
 * both F32, F16 or BF16, nb[0] = the element size, receive rows 0 .. n - 1 of
 * every set; rows at or past len[s] (int32 [Bk], device) become zeros.
 * E.g. a cached prefix for a dense attention call, or a cache to be saved.
 */
ACEFA_API int acefa_kv8_load(const acefa_kv8_cache *cache, const int32_t *len, const acefa_tensor *k_dst,
                             const acefa_tensor *v_dst, void *stream);

/*
 * Attention of a few new tokens per set over the cache (a decode step, or a
 * handful of drafted tokens), after their rows were stored.
 *   q       [D, n_q, Hq, Bk] F32, F16 or BF16, nb[0] = the element size;
 *           Hq % Hkv == 0 and n_q * Hq / Hkv <= ACEFA_KV8_MAX_ROWS (longer
 *           prompts: acefa_flash_attn_packed on their own K and V)
 *   len     int32 [Bk], device: rows in each set, the new ones included
 *           (values outside [0, n_max] count as the nearer bound)
 *   dst     [D, Hq, n_q, Bk] F32, F16 or BF16, nb[0] = the element size
 *   weight  F32 [n_max, Hkv, Bk], nb[0] == 4, or NULL
 * Query i sees rows j < len - (n_q - 1 - i) of its set.  dst = softmax(scale *
 * q k^T) v; a query that sees nothing gives 0, and a block whose scale is NaN
 * reaches only the queries that see one of its rows.  dst and weight lie apart
 * from one another, from q and from the cache.  With `weight`, weight[j, h, s]
 * grows by the softmax weights of row j summed over the n_q * Hq / Hkv
 * queries of its head -- what acefa_kv8_evict goes by; rows at or past
 * len[s] are left alone.  Q enters whole and all sums are F32.  The softmax
 * weights that multiply V are rounded to 22 bits, or to 11 (F16) where q and dst
 * both have 16-bit types, and to steps of 2^-32 of the row's largest; those that
 * `weight` receives are F32 (a NaN in q makes those of its head NaN).
 * Results do not depend on the order in which the GPU runs the blocks.
 * workspace: acefa_kv8_attn_workspace_bytes(), 256-B aligned, no
 * initialisation; a function of shapes and the device only.  Calls that may
 * overlap on the GPU need a workspace each.
 */
#define ACEFA_KV8_MAX_ROWS 64
ACEFA_API int acefa_kv8_attn(const acefa_tensor *q, const acefa_kv8_cache *cache, const int32_t *len,
                             const acefa_tensor *dst, float scale, const acefa_tensor *weight, void *stream,
                             void *workspace, size_t workspace_bytes);
/* 0 for operands that acefa_kv8_attn refuses, or without a device. */
ACEFA_API size_t acefa_kv8_attn_workspace_bytes(const acefa_tensor *q, const acefa_kv8_cache *cache,
                                                const acefa_tensor *weight);

/*
 * Eviction: each (head, set) of `cache` keeps `keep` = kept->ne[0] of its rows
 * in `out`, in their order.
 *   weight      F32 [n_max, Hkv, Bk]: accumulated attention weights
 *   len         int32 [Bk], device: rows in each set
 *   n_first, n_recent  the first and the last rows that are kept whatever
 *               their weight (n_first + n_recent <= keep)
 *   out         the cache of the rows that stay, keep <= its n_max, same D, Hkv
 *               and Bk; must not overlap `cache`.  Rows behind keep stay as they
 *               are: with a longer n_max acefa_kv8_store goes on at len_out (with
 *               n_max == keep a set that was shrunk is full)
 *   kept        I32 [keep, Hkv, Bk], nb[0] == 4: the kept rows, ascending
 *   weight_out  F32 [keep, Hkv, Bk], nb[0] == 4, or NULL: their weights (also as
 *               the first rows of an [n_max, Hkv, Bk] array for acefa_kv8_attn,
 *               whose rows behind keep the caller clears before it goes on)
 *   len_out     int32 [Bk], device: min(len, keep)
 * The other places go to the largest weights, equal ones to the lower row
 * (-0 equals 0; a NaN ranks below every number).  A set of at most keep rows
 * keeps them all.  A block of `out` takes the largest scale of the rows that
 * come into it; rows of that scale move unchanged, the others become
 * q * d_old / d rounded once to the nearest integer, ties to even.  A NaN scale
 * counts as the largest, and all rows that meet it move unchanged.  Behind
 * len_out, up to keep, `kept` is -1 and rows, scales of blocks without a row
 * and weight_out are 0.
 */
ACEFA_API int acefa_kv8_evict(const acefa_kv8_cache *cache, const acefa_tensor *weight, const int32_t *len,
                              int64_t n_first, int64_t n_recent, const acefa_kv8_cache *out,
                              const acefa_tensor *kept, const acefa_tensor *weight_out, int32_t *len_out,
                              void *stream);

/*
 * Attention of whole sequences packed behind one another: the prompts of
 * several requests, or the texts of several captions, in one call with no
 * padding.  The reference prefills one sequence per call
 * (src/pipeline-lm.cpp:317-344).
 *   q     [D, rows_q,  Hq,  1] F16 or BF16, D 64 or 128
 *   k, v  [D, rows_kv, Hkv, 1] of q's type; Hq % Hkv == 0
 *   dst   [D, Hq, rows_q, 1] of q's type or F32
 *   cu_q, cu_k  int32 [n_seq + 1], device: sequence s is rows cu_q[s] ..
 *         cu_q[s + 1] - 1 of q and cu_k[s] .. cu_k[s + 1] - 1 of k and v
 *         (cu_k NULL: cu_q); sequences may be empty
 *   mask  0: every query sees every key of its sequence; ACEFA_MASK_CAUSAL:
 *         query i of n_q sees key j <= i + n_k - n_q (a prompt, or the last
 *         n_q tokens of one); ACEFA_MASK_WINDOW: |i - j| <= window
 * dst = softmax(scale * q k^T) v per sequence, scale > 0, sums in F32; the weights
 * that multiply v are rounded to the operands' type (11 bits, in steps of 2^-32 of
 * the row's largest, or BF16's 8), their sum takes them whole.  A query
 * that sees nothing gives 0.  Rows of dst outside every sequence are left as
 * they were, and rows of k and v outside a sequence never reach it, whatever
 * they hold; a NaN or an infinity in a sequence's own v may reach every query of
 * that sequence and head.  Offsets must not decrease: a sequence whose offsets do, or leave
 * the tensors, is left unwritten and raises device error 5 (acefa_device_error());
 * where cu_q decreases, so are all sequences behind.  nb[0] = the element size; data and nb[1..2] of q, k and
 * v multiples of 16 bytes, not 0; dst aligned to its elements, its rows apart, and
 * apart from q, k and v (in one buffer with them only where all rows are the same
 * distance apart).  rows_q and rows_kv up to 2^24, n_seq <= 65535,
 * Hq <= 4096.  No workspace.
 */
ACEFA_API int acefa_flash_attn_packed(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                      const acefa_tensor *dst, const int32_t *cu_q, const int32_t *cu_k, int n_seq,
                                      int mask, int window, float scale, void *stream);

/* Workspace acefa_flash_attn_ext() needs for these operands on the current device
 * (dense path only: mask tile classes, the partial results of the last-wave
 * key-range split, and for BF16 K/V F16 copies of K and V, 4 bytes per K/V
 * value; decode nodes need a token 256 bytes).  A function of shapes,
 * types and the device only -- never of tensor contents -- so it can be sized
 * once before CUDA-graph capture.  A smaller workspace also works where the
 * operator can do without: it then skips the BF16 copies (converting inside
 * the attention kernel, same results) and splits fewer key ranges.  Returns 0
 * for unsupported operands. */
ACEFA_API size_t acefa_workspace_bytes(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                                       const acefa_tensor *mask, const acefa_tensor *dst);

/* 1 if acefa_flash_attn_ext accepts these operands, else 0 (mirrors
 * ggml_backend_cuda_device_supports_op for GGML_OP_FLASH_ATTN_EXT; when it
 * returns 0 the ggml scheduler keeps the node on the CPU backend). */
ACEFA_API int acefa_supports(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                             const acefa_tensor *mask, const acefa_tensor *sinks, const acefa_tensor *dst);

/* Validation only: the status acefa_flash_attn_ext would return before
 * launching (ACEFA_OK when the operands are accepted).  Touches no device. */
ACEFA_API int acefa_check(const acefa_tensor *q, const acefa_tensor *k, const acefa_tensor *v,
                          const acefa_tensor *mask, const acefa_tensor *sinks, const acefa_tensor *dst);

/* Reads and clears the device-side error word set by bounded waits inside the
 * kernels (0 = none).  Synchronises `stream`; for diagnostics, not hot paths.
 * There is ONE word per device, shared by every stream and thread using the
 * engine on it: the first code recorded since the last read is kept, whichever
 * call's kernel recorded it, and a read from one stream also clears what a
 * kernel on another stream recorded.  Callers that run the engine on several
 * streams of one device and need to know which call failed read it with those
 * streams idle.  Returns a negative acefa_status if the read itself fails. */
ACEFA_API int acefa_device_error(void *stream);

/* Human-readable name of an acefa_status. */
ACEFA_API const char *acefa_status_string(int status);

/* Kernel-launch count of the last successful call on this host thread:
 * acefa_flash_attn_ext 1 to 3 (mask classification, attention, split-KV
 * combine), acefa_flash_attn_packed, acefa_kv8_store and acefa_kv8_load 1,
 * acefa_kv8_attn 1 or 2, acefa_kv8_evict 2; calls without rows 0. */
ACEFA_API int acefa_last_launch_count(void);

/* Which kernel family served the last successful attention call on this thread
 * (acefa_kv8_store, _load, _evict and calls without rows leave it as it was):
 * 1 = split-KV decode (mma.sync), 2 = dense tcgen05/TMEM, 3 = packed sequences
 * (tcgen05/TMEM, few rows mma.sync), 4 = decode over an 8-bit block-scaled cache. */
ACEFA_API int acefa_last_path(void);

/* ABI version: major*10000 + minor*100 + patch. */
ACEFA_API int acefa_version(void);

#ifdef __cplusplus
}
#endif
#endif /* ACEFA_H */
