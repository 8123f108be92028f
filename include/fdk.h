/*
 * fdk - flash-decode kernels for MI355X (gfx950): C ABI.
 *
 * One hot path: split-KV GQA decode attention over a paged KV cache plus the log-sum-exp
 * combine of the per-split partials.  Plain C: raw device pointers, element strides, sizes,
 * a HIP stream handle passed as void*.  No C++ or torch types cross this boundary.
 *
 * What each entry point stands in for in the reference (paths relative to the reference root;
 * the reference's own FFI for this path is the Triton AOT launcher
 *   CUresult <kernel>_ex(CUstream, <pointers / i32 / fp32 in kernel-argument order>, algo_info)
 * generated by python/triton_dist/tools/compile_aot.py:330-333,405-435 and called from
 * python/triton_dist/kernels/nvidia/flash_decode.py:1075-1089):
 *
 *   fdk_decode           gqa_fwd_batch_decode_intra_rank / _aot, flash_decode.py:847-928, 1037-1092
 *                        (split launch + combine launch; packed [B,Hq,D+1] result when pack_lse=1)
 *                        and gqa_fwd_batch_decode, :763-844 (out only).
 *   fdk_decode_splitkv   distributed.gqa_fwd_batch_decode_split_kv_*  (kernel :129-239, call :1075-1086)
 *   fdk_combine          distributed.intra_rank_gqa_fwd_batch_decode_combine_kv_* (kernel :392-449,
 *                        call :1087-1089) and gqa_fwd_batch_decode_combine_kv_* (:307-360)
 *   fdk_combine_ranks    distributed.inter_rank_gqa_fwd_batch_decode_combine_kv_* (kernel :481-532,
 *                        call layers/nvidia/sp_flash_decode_layer.py:164-183)
 *   fdk_plan             get_triton_split_kv_algo_info / get_triton_combine_kv_algo_info,
 *                        flash_decode.py:103-109, 281-285 (the constants a launch is specialised on;
 *                        here the split count is chosen from the shape instead of fixed at 32, :863)
 *   fdk_workspace_bytes  the ``output_split`` allocation, flash_decode.py:867-868
 *   fdk_counters_len     sizes the counters of the single-launch / work-queue form; the reference's counterpart is the
 *                        ``workspace`` int32 tensor of its persistent kernel (flash_decode.py:931-976,
 *                        test_decode_attn.py:150)
 *   fdk_last_error       the launcher's fprintf(stderr) diagnostics, compile_aot.py:426-434
 *   fdk_kv_append        the step before the path: rmsnorm_rope_update_kv_cache_task_compute,
 *                        mega_triton_kernel/kernels/norm.py:32-190, built by
 *                        ModelBuilder.make_qk_norm_rope_update_kvcache, models/model_builder.py:341-379
 *                        (per-head RMSNorm of q and k, rotary embedding, K/V rows appended to the paged cache)
 *
 * Without a counterpart in the reference (revision 3):
 *   fdk_kv_append_axes   the append with explicit positions of one to four axes, and into MXFP4 caches
 *   fdk_mx_quantize, fdk_mx_dequantize    16-bit rows to and from MXFP4 rows
 *   fdk_accumulate_weights                what each cached token receives from a query's attention
 *   fdk_kv_evict, fdk_kv_evict_workspace_bytes    the tokens with the least of it leave the cache
 *
 * Conventions
 *   - Return value: 0 on success; a negative FDK_E* code when the arguments are rejected (nothing was
 *     launched); a positive value is the hipError_t of a failed launch.  Never exits the process.
 *   - All launches are asynchronous on the given stream; no host synchronisation, no device allocation,
 *     no host read of device data.  Safe to call from several host threads.  The library keeps no
 *     mutable state apart from a thread-local error string (and a cache of the device's CU count).
 *   - The caller owns every buffer.  Scratch memory for the split partials comes in through
 *     ``workspace`` (size from fdk_workspace_bytes).
 *   - Strides are in ELEMENTS of the respective tensor's dtype.  The head dimension is contiguous.
 *   - Token n of sequence b lives at pool row  block_table[b, n / page_size] * page_size + n % page_size
 *     (flash_decode.py:203-205).  Any of the max_pages columns of a row may be read (the whole row must be
 *     addressable memory), but an entry past ceil(kv_len/page_size) is never used as a page number: its
 *     value does not matter and nothing is loaded through it.
 *   - lse is the natural-log log-sum-exp of the scaled (and soft-capped) logits, out is normalised by
 *     the local softmax sum: exactly what the reference's cross-rank combine consumes (:512-526).
 *   - A sequence with kv_len == 0 yields out = 0 and lse = -inf (the reference yields NaN there, :441-449).
 */
#ifndef FDK_H_
#define FDK_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Compatibility.  FDK_ABI_VERSION names a line of layouts and changes only when a caller compiled against an older
 * header of the same version would stop working.  Within a version the argument structs only grow at the end:
 * struct_size tells the library which fields the caller knows, fields past it read as zero, and FDK_ABI_REVISION
 * counts the additions (fdk_abi_revision() is the library's).  A caller built against revision 0 of version 8
 * runs unchanged against this library; a caller whose struct is LARGER than the library's is refused (FDK_EABI). */
#define FDK_ABI_VERSION 8
#define FDK_ABI_REVISION 3

typedef enum fdk_dtype {
    FDK_BF16 = 0,
    FDK_FP16 = 1,
    FDK_FP8_E4M3 = 2, /* OCP e4m3fn, KV cache only */
    FDK_FP32 = 3,     /* partials / packed-rank buffers only */
    FDK_MXFP4 = 4     /* (revision 3) KV cache only: OCP microscaling rows of 4-bit values.  A row of D values is D/2 bytes of
                         e2m1 codes (value 2i in the low four bits of byte i) and, in a tensor of its own, D/32 e8m0 bytes,
                         one per block of 32 consecutive values: value = code * 2^(byte - 127), byte 255: NaN.  Strides of
                         both are in bytes */
} fdk_dtype;

typedef enum fdk_status {
    FDK_OK = 0,
    FDK_ENULL = -1,        /* a required pointer is null */
    FDK_EALIGN = -2,       /* pointer or stride not 16-byte aligned */
    FDK_ESHAPE = -3,       /* inconsistent or out-of-range dimension */
    FDK_EUNSUPPORTED = -4, /* dtype / head_dim / algorithm combination not built */
    FDK_EWORKSPACE = -5,   /* workspace missing or too small */
    FDK_EABI = -6          /* struct_size is smaller than the first revision's or larger than this library's */
} fdk_status;

typedef enum fdk_algo {
    FDK_ALGO_AUTO = 0,
    FDK_ALGO_VALU = 1, /* v_dot2 / FMA path, any group size */
    FDK_ALGO_MFMA = 2  /* matrix-core path (group padded to 16 rows) */
} fdk_algo;

/* Launch plan: the shape-dependent constants of one decode call. */
typedef struct fdk_plan_t {
    int32_t num_splits;   /* S >= 1: the workspace holds S partial rows per (sequence, q head);
                             S == 1: no workspace, fdk_decode writes the result in one pass.
                             Chunk mode: also the grid extent over the KV axis */
    int32_t chunk_tokens; /* chunk mode: tokens per split; split s of sequence b covers
                             [s*chunk, min((s+1)*chunk, kv_len[b])) (the last split: to kv_len[b]); a multiple
                             of 16, of 64 for a forced split count.  With chunk_floor > 0: the most a split holds.
                             Balanced mode: nominal tokens per workgroup (informational) */
    int32_t algo;         /* resolved fdk_algo */
    int32_t kv_heads_per_wg; /* matrix-core path: adjacent kv heads one workgroup reads */
    int32_t balanced;     /* 1: balanced mode - the kernel reads kv_lens and cuts the KV ranges of the
                             whole batch into `workgroups` equal shares (ragged batches stay balanced);
                             0: chunk mode - every sequence is cut into num_splits chunks */
    int32_t workgroups;   /* balanced mode: workgroups of the split kernel */
    int32_t chunk_floor;  /* chunk mode, > 0: the chunks follow each sequence's own length (as the reference's
                             cdiv(kv_len, NUM_KV_SPLITS), flash_decode.py:151-153): sequence b is cut every
                             clamp(ceil(kv_len[b] / num_splits) rounded up to 16, chunk_floor, chunk_tokens)
                             tokens.  Chosen (matrix-core path) when the host has not said that the lengths are
                             alike (min_kv_len), also for a forced split count */
    int32_t reserved;
} fdk_plan_t;

typedef struct fdk_decode_args {
    uint32_t struct_size; /* = sizeof(fdk_decode_args) of the header the caller was compiled with */
    uint32_t flags;       /* FDK_FLAG_* */

    /* query [B, Hq, D], D = head_dim */
    const void* q;
    int64_t q_stride_b, q_stride_h;
    int32_t q_dtype; /* FDK_BF16 | FDK_FP16 */

    /* caches [num_pages, P, Hkv, D] (v_cache: Dv, see v_head_dim); strides of the page, token-in-page and head axes */
    int32_t kv_dtype; /* q_dtype | FDK_FP8_E4M3 | FDK_MXFP4 (rows of D/2 bytes, strides in bytes) */
    const void* k_cache;
    const void* v_cache;
    int64_t k_stride_page, k_stride_tok, k_stride_head;
    int64_t v_stride_page, v_stride_tok, v_stride_head;
    const float* k_scale; /* [Hkv] dequantisation scales, FDK_FP8_E4M3 only (null = 1.0).  On the matrix-core path a K scale
                             that is a power of two (1.0 among them) costs nothing: it is the exponent operand of the
                             conversion, which is the exact k8 * scale */
    const float* v_scale;

    const int32_t* block_table; /* [B, max_pages] */
    int64_t table_stride_b;
    const int32_t* kv_lens; /* [B] */

    int32_t batch, num_q_heads, num_kv_heads, head_dim;
    int32_t page_size;
    int32_t max_pages;  /* columns of block_table; max_pages * page_size <= 2^30 tokens */
    int32_t max_kv_len; /* host-known upper bound of kv_lens (0: max_pages*page_size).  It sizes the plan only: a
                           value that is too small costs balance, never tokens (the last split runs to kv_len) */
    int32_t min_kv_len; /* host-known lower bound of kv_lens (0: unknown).  When it is within 1/32 of the upper bound
                           the lengths are taken to be alike: whole sequences per workgroup (a single pass, no combine
                           launch) where they fill the GPU, per-sequence chunks of one size otherwise.  Unknown or far
                           apart: long contexts of two or more sequences are cut into equal shares of the tokens that
                           kv_lens holds (balanced mode), because whole sequences per workgroup are as slow as the
                           longest one, and per-sequence chunks follow each sequence's own length (chunk_floor of the
                           plan).  Like max_kv_len it never changes results */
    int32_t num_splits; /* 0: choose; >0: force this many splits */

    float sm_scale;
    float soft_cap; /* <= 0: off */

    /* results */
    void* out; /* [B, Hq, Dv] (or [B, Hq, Dv+1] when FDK_FLAG_PACK_LSE), dtype out_dtype; Dv = head_dim unless v_head_dim says otherwise */
    int64_t out_stride_b, out_stride_h;
    int32_t out_dtype;  /* FDK_BF16 | FDK_FP16 | FDK_FP32 */
    int32_t algo;       /* fdk_algo */
    float* lse;         /* [B, Hq] fp32, may be null */
    int64_t lse_stride_b;

    /* scratch for split partials: fp32 o [B,Hq,S,D] followed by fp32 lse [B,Hq,S] */
    void* workspace;
    size_t workspace_bytes;

    /* Optional: fdk_counters_len(args) int32 counters that are ZERO on entry (matrix-core path).  With them
     *   - a forced split count with more pieces than fit the GPU at once runs as a fixed set of workgroups that pull
     *     the pieces from a queue, so ragged batches keep every compute unit busy to the end;
     *   - with FDK_FLAG_SINGLE_LAUNCH a call whose plan splits the KV range is ONE launch (see the flag).
     * Every call leaves the counters zero again.  Calls that overlap in time need distinct counters.
     * Null: one workgroup per piece, then the combine kernel. */
    int32_t* counters;
    int64_t counters_len;

    /* Reserved; set to 0.  (The first revision of this layout carried measurement overrides here.  They changed
     * timing only; the library ignores them now, so a caller compiled against that revision keeps working.) */
    int32_t reserved0[4];

    /* Optional length feedback for callers whose kv_lens exist only on the GPU (the reference's entry points take
     * nothing else): 4 int32 that the GPU can write, 16-byte aligned - device memory, or host memory mapped for the
     * GPU (fdk_length_feedback_alloc).  The call stores {min_b n_b, max_b n_b, epoch, batch} there, n_b = kv_lens[b]
     * clamped to [0, max_pages * page_size], epoch = a per-process call count (never 0).  Read it before a LATER call
     * on the same batch and pass what it holds as min_kv_len / max_kv_len: the bounds only size the plan, so a value
     * that is out of date costs time, never tokens.  Written by one wavefront of the last kernel of the call.
     * Null: nothing is stored. */
    int32_t* length_feedback;

    /* Reserved; set to 0 (first revision: a measurement buffer and its length; ignored). */
    void* reserved1;
    int64_t reserved2;

    /* ---- fields added after the first revision of this layout (struct_size tells the library which exist) ---- */

    /* Null in product use.  Measurement overrides and probes of the benchmark (include/fdk_measure.h). */
    const struct fdk_measure_args* measure;

    /* (revision 2) Values per V row and per output row where they differ from head_dim, which then counts the values
     * of a q and K row only - the reference's V_DIM / BLOCK_DV next to K_DIM (flash_decode.py:103-109,170-177): 0 =
     * head_dim.  Built: head_dim 64, 128, 256 with v_head_dim = head_dim (every path), and on the matrix-core path
     * (16-bit and e4m3 caches) head_dim 192 (a row of 128 + 64 values, the reference's BLOCK_HEAD_DIM + BLOCK_DPE) with
     * v_head_dim 192 or 128, and head_dim 576 (512 + 64) with v_head_dim 512.  out, lse, the packed row and the workspace
     * follow v_head_dim: out is [B, Hq, Dv], the packed lse sits at out[b, h, Dv], fdk_workspace_bytes takes Dv. */
    int32_t v_head_dim;
    int32_t reserved3;

    /* (revision 3) kv_dtype FDK_MXFP4: the scale bytes of the caches, [num_pages, P, Hkv, D/32], with byte strides of the
     * page, token and head axes; rows aligned to 4 bytes (head_dim 64: 2).  k_scale / v_scale are not read.  Built for
     * head_dim 64, 128 and 256 with v_head_dim = head_dim on the matrix-core path; no single-launch form; with counters, too, a forced split count runs as
     * one workgroup per piece.  A value takes part as code * 2^(byte - 127) converted to q's dtype, exact within its range (a
     * cache written for bf16 and read with fp16 queries may hold values beyond 65504: infinities, and NaN where they are weighed) */
    const uint8_t* k_block_scale;
    const uint8_t* v_block_scale;
    int64_t kbs_stride_page, kbs_stride_tok, kbs_stride_head;
    int64_t vbs_stride_page, vbs_stride_tok, vbs_stride_head;
} fdk_decode_args;

#define FDK_FLAG_PACK_LSE 1u /* also store lse, converted to out_dtype, at out[b, h, D] (flash_decode.py:446-449) */
#define FDK_FLAG_DRY_RUN 2u  /* validate and plan only; touch no device, launch nothing */
#define FDK_FLAG_SINGLE_LAUNCH 8u /* with args->counters: no combine launch - the workgroup that is last to finish a
                                     piece of a (sequence, head block, head tile) merges the pieces into (out, lse)
                                     itself: the single-launch form of the reference's persistent kernel
                                     (flash_decode.py:587-760) without its grid barrier.  The pieces cross the XCDs'
                                     separate L2 caches, so they are written through and read around them; on
                                     MI355X that costs more than the second launch saves - off unless asked for */
#define FDK_FLAG_FP8_FOLD_K_SCALE 16u /* fp8 cache, matrix-core path: logits are (q . k8) * k_scale instead of
                                         q . round_to_q_dtype(k8 * k_scale).  The default reproduces a decode over the
                                         dequantised cache exactly, which costs a conversion to fp32, a multiplication
                                         and a re-packing per K value; folded, the values are converted exactly and the
                                         scale is applied to the logits (the form serving engines use).  The two differ
                                         by the rounding of the dequantised K to 16 bits (relative 2^-9 per element;
                                         about 1e-3 in a logit of 128 unit-variance terms): inside the tolerances of
                                         this path for long diffuse contexts, not for a softmax that one or a few
                                         tokens dominate.  V is converted exactly and scaled once in either form.
                                         Ignored by the vector path */
/* bit 4u is reserved (first revision: a measurement probe, now fdk_measure_args.probe_loads); it is ignored */

/* Cross-rank merge arguments: partial [R, B, Hq, D(+1)] + lse, kv_lens [R, B]. */
typedef struct fdk_combine_ranks_args {
    uint32_t struct_size;
    uint32_t flags;          /* FDK_FLAG_PACK_LSE: lse of rank r is read from partial[r,b,h,D] */
    const void* partial;     /* [R, B, Hq, D] or [R, B, Hq, D+1] */
    int64_t stride_r, stride_b, stride_h;
    int32_t partial_dtype;   /* FDK_BF16 | FDK_FP16 | FDK_FP32 */
    int32_t out_dtype;
    const float* partial_lse; /* [R, B, Hq] fp32 when not packed */
    int64_t lse_stride_r, lse_stride_b;
    const int32_t* kv_lens;  /* [R, B]; rank r contributes to b iff kv_lens[r,b] > 0 */
    int32_t num_ranks, batch, num_q_heads, head_dim;
    void* out;               /* [B, Hq, D] */
    int64_t out_stride_b, out_stride_h;
    float* lse;              /* [B, Hq] fp32 merged lse, may be null */
    int64_t lse_stride_b_out;
} fdk_combine_ranks_args;

/* Per-head RMSNorm + rotary embedding of the new tokens' q and k rows, and the append of their K / V rows to
 * the paged cache.  kv_lens already counts the new tokens: token t (0 <= t < new_tokens) of sequence b sits at
 * position pos = kv_lens[b] - new_tokens + t, i.e. at cache row block_table[b, pos / page_size] * page_size +
 * pos % page_size (the row the decode kernels read; the reference kernel omits the page_size factor,
 * norm.py:115,183, which is the same only for page_size 1).
 *   q, k rows  y = w * (x * rsqrt(mean(x^2) + eps)) in fp32, halves rounded to the 16-bit dtype, then
 *              (y0, y1) -> (y0 cos - y1 sin, y1 cos + y0 sin) with y0 = y[:D/2], y1 = y[D/2:] and the first D/2
 *              columns of row pos of the fp32 cos / sin tables (norm.py:127-171)
 *   v rows     copied
 * An fp8 cache (kv_dtype = FDK_FP8_E4M3) receives clamp(x16 / scale[h], -448, 448) rounded to nearest even,
 * x16 being the 16-bit value a 16-bit cache would have received.  Positions outside [0, max_pages * page_size)
 * and table entries outside [0, num_pages) are not written.  A token's cos / sin row index is clamped to
 * [0, max_positions). */
typedef struct fdk_kv_append_args {
    uint32_t struct_size; /* = sizeof(fdk_kv_append_args) */
    uint32_t flags;       /* FDK_FLAG_DRY_RUN */
    const void* qkv;      /* [B, T, Hq + 2 Hkv, D]: q heads, then k heads, then v heads */
    int64_t qkv_stride_b, qkv_stride_t, qkv_stride_h;
    int32_t qkv_dtype;    /* FDK_BF16 | FDK_FP16 (also of the weights and of q_out) */
    int32_t kv_dtype;     /* = qkv_dtype, or FDK_FP8_E4M3 (fdk_kv_append_axes: also FDK_MXFP4) */
    const void* q_weight; /* [D] RMSNorm weight of the q heads */
    const void* k_weight; /* [D] RMSNorm weight of the k heads */
    float q_eps, k_eps;
    const float* cos;     /* [1 or B, max_positions, >= D/2 columns] fp32, row = absolute position */
    const float* sin;
    int64_t cs_stride_b;  /* 0: one table for all sequences */
    int64_t cs_stride_pos;
    int32_t max_positions;
    int32_t batch, new_tokens, num_q_heads, num_kv_heads, head_dim;
    const int32_t* block_table; /* [B, max_pages] */
    int64_t table_stride_b;
    const int32_t* kv_lens;     /* [B], lengths after the append */
    int32_t page_size, max_pages, num_pages;
    void* k_cache;        /* [num_pages, page_size, Hkv, D] */
    void* v_cache;
    int64_t k_stride_page, k_stride_tok, k_stride_head;
    int64_t v_stride_page, v_stride_tok, v_stride_head;
    const float* k_scale; /* [Hkv] fp32, fp8 caches only */
    const float* v_scale;
    void* q_out;          /* [B, T, Hq, D] */
    int64_t q_out_stride_b, q_out_stride_t, q_out_stride_h;
} fdk_kv_append_args;

/* (revision 3) The append with explicit positions, and into an MXFP4 cache: the block of fdk_kv_append and what it lacks.
 *   Positions: pair i of a row (y[i], y[i + D/2]) turns by row positions[axis(i), b, t] of the cos / sin tables instead of row
 * pos - a cache from which tokens were evicted, where a token's place is not its position, or positions of several axes
 * (time, height, width).  rope_sections[x] pairs belong to axis x and add up to D/2: one section after the other, or, with
 * rope_interleaved, pair i to axis i mod num_axes while i / num_axes < rope_sections[that axis] and to axis 0 otherwise.
 * Where K / V rows go is still decided by kv_lens.
 *   MXFP4 (append->kv_dtype = FDK_MXFP4): the caches' rows are D/2 bytes with strides in bytes, 2-byte aligned; they receive
 * the codes and scales that fdk_mx_quantize gives for the 16-bit values a 16-bit cache would have received. */
typedef struct fdk_kv_append_axes_args {
    uint32_t struct_size;     /* = sizeof(fdk_kv_append_axes_args) */
    uint32_t flags;           /* FDK_FLAG_DRY_RUN (here or in *append) */
    const fdk_kv_append_args* append;
    const int32_t* positions; /* [num_axes, B, T], strides in elements; null: the tokens' places in the cache */
    int64_t pos_stride_axis, pos_stride_b, pos_stride_t;
    int32_t num_axes;         /* 1 .. 4 (0 without positions) */
    int32_t rope_interleaved;
    int32_t rope_sections[4];
    uint8_t* k_block_scale;   /* FDK_MXFP4: [num_pages, P, Hkv, D/32], byte strides of the page, token and head axes */
    uint8_t* v_block_scale;
    int64_t kbs_stride_page, kbs_stride_tok, kbs_stride_head;
    int64_t vbs_stride_page, vbs_stride_tok, vbs_stride_head;
} fdk_kv_append_axes_args;

/* (revision 3) Conversion between 16-bit rows and MXFP4 rows (see FDK_MXFP4): n0 x n1 x n2 rows of num_values values, each
 * tensor with strides of its three row axes (elements; bytes for codes and scales), values contiguous.
 *   fdk_mx_quantize    writes codes and scales: the scale of a block is the smallest power of two with amax <= 7 scales,
 *                         within [2^-126, 2^125] for bf16 and [2^-126, 2^13] for fp16 (so that 6 scales are finite in the
 *                         type); codes are rounded to nearest, ties to even, and saturate at 6.  A block that holds an
 *                         infinity or a NaN gets scale byte 255
 *   fdk_mx_dequantize  writes x: code * 2^(byte - 127) in x_dtype */
typedef struct fdk_mxfp4_args {
    uint32_t struct_size;
    uint32_t flags;       /* FDK_FLAG_DRY_RUN */
    void* x;              /* FDK_BF16 | FDK_FP16, 16-byte aligned rows */
    uint8_t* codes;       /* 4-byte aligned rows of num_values / 2 bytes */
    uint8_t* scales;      /* rows of num_values / 32 bytes */
    int64_t x_stride[3], codes_stride[3], scales_stride[3];
    int32_t n[3];
    int32_t num_values;   /* a positive multiple of 32 */
    int32_t x_dtype;
    int32_t reserved;
} fdk_mxfp4_args;

/* (revision 3) Attention weights per cached token, for the eviction of those that receive little:
 *   weights[b, kvh, n] += sum over the q heads h of kv head kvh of exp(logit(b, h, n) - lse[b, h]),  n < kv_lens[b],
 * logit being the scaled (and soft-capped) logit of the decode and lse what it returned.  K rows of 64, 128, 192, 256 or 576
 * values (MXFP4: 64, 128, 256).  Lengths are clamped to weights_len and to the table.  Nothing else is written. */
typedef struct fdk_attn_weights_args {
    uint32_t struct_size;
    uint32_t flags;       /* FDK_FLAG_DRY_RUN */
    const void* q;        /* [B, Hq, D] */
    int64_t q_stride_b, q_stride_h;
    int32_t q_dtype;      /* FDK_BF16 | FDK_FP16 */
    int32_t kv_dtype;     /* q_dtype | FDK_FP8_E4M3 | FDK_MXFP4 */
    const void* k_cache;  /* [num_pages, P, Hkv, D] */
    int64_t k_stride_page, k_stride_tok, k_stride_head;
    const float* k_scale; /* [Hkv], fp8 caches only (null = 1.0) */
    const uint8_t* k_block_scale; /* MXFP4 caches: [num_pages, P, Hkv, D/32], byte strides */
    int64_t kbs_stride_page, kbs_stride_tok, kbs_stride_head;
    const int32_t* block_table; /* [B, max_pages] */
    int64_t table_stride_b;
    const int32_t* kv_lens;     /* [B] */
    const float* lse;           /* [B, Hq] */
    int64_t lse_stride_b;
    float* weights;             /* [B, Hkv, weights_len], updated in place */
    int64_t weights_stride_b, weights_stride_h;
    int32_t batch, num_q_heads, num_kv_heads, head_dim;
    int32_t page_size, max_pages, weights_len;
    float sm_scale, soft_cap;   /* soft_cap <= 0: off */
    int32_t reserved;
} fdk_attn_weights_args;

/* (revision 3) Eviction.  Of a sequence's n = kv_lens[b] tokens (clamped to weights_len and to the table) the last `recent`
 * stay and, of the others, those with the largest weights - ties: the lowest slots; a NaN counts as the largest -, `keep` in
 * all; every kv head chooses for itself.  The survivors' rows move to slots 0 .. in their order, in place; rows behind the new
 * length keep their contents, pages of the table keep their owners.  A sequence of at most `keep` tokens stays as it is.
 *   kept[b, kvh, j]  the slot that the token in slot j had before, -1 behind the new length
 *   weights_out      the survivors' weights, 0 behind them; may be `weights` itself (same strides), no other overlap
 *   kv_lens_out      min(n, keep); may be `kv_lens` itself */
typedef struct fdk_kv_evict_args {
    uint32_t struct_size;
    uint32_t flags;       /* FDK_FLAG_DRY_RUN */
    int32_t kv_dtype;     /* FDK_BF16 | FDK_FP16 | FDK_FP8_E4M3 | FDK_MXFP4 */
    int32_t reserved0;
    void* k_cache;        /* [num_pages, P, Hkv, D], rows of a multiple of 16 bytes */
    void* v_cache;        /* [num_pages, P, Hkv, Dv]; may be a part of the K rows (same strides), which then move once */
    int64_t k_stride_page, k_stride_tok, k_stride_head;
    int64_t v_stride_page, v_stride_tok, v_stride_head;
    uint8_t* k_block_scale; /* MXFP4 caches: the scales move with the rows; byte strides */
    uint8_t* v_block_scale;
    int64_t kbs_stride_page, kbs_stride_tok, kbs_stride_head;
    int64_t vbs_stride_page, vbs_stride_tok, vbs_stride_head;
    const int32_t* block_table; /* [B, max_pages] */
    int64_t table_stride_b;
    const int32_t* kv_lens;     /* [B] */
    const float* weights;       /* [B, Hkv, weights_len] */
    int64_t weights_stride_b, weights_stride_h;
    float* weights_out;         /* [B, Hkv, weights_len] */
    int64_t weights_out_stride_b, weights_out_stride_h;
    int32_t* kept;              /* [B, Hkv, keep], contiguous */
    int32_t* kv_lens_out;       /* [B] */
    void* workspace;            /* fdk_kv_evict_workspace_bytes, 16-byte aligned; contents unspecified before and after */
    size_t workspace_bytes;
    int32_t batch, num_kv_heads, head_dim, v_head_dim; /* v_head_dim 0: head_dim */
    int32_t page_size, max_pages, weights_len;
    int32_t keep, recent;       /* 0 <= recent <= keep, 1 <= keep <= weights_len */
    int32_t num_pages;          /* of the pool: rows of pages outside it are left out */
} fdk_kv_evict_args;

struct fdk_measure_args; /* include/fdk_measure.h */

int fdk_abi_version(void);
int fdk_abi_revision(void);

/* Message for the last non-zero return on the calling thread ("" if none). */
const char* fdk_last_error(void);

/* Number of compute units the plan heuristics assume for the current device (256 when no device
 * can be queried). */
int fdk_device_cus(void);

/* Fill *plan for these arguments (uses batch, heads, head_dim, strides, page_size, max_pages, the length
 * hints max_kv_len / min_kv_len, num_splits, algo).  num_cus <= 0: query the current device.  Touches no
 * device memory. */
int fdk_plan(const fdk_decode_args* args, int num_cus, fdk_plan_t* plan);

/* Bytes of workspace that hold the partials of ``num_splits`` splits.  fdk_decode needs it only when
 * its plan has more than one split; fdk_decode_splitkv / fdk_combine always do.  head_dim: the values of an output
 * row (v_head_dim where the call sets one). */
size_t fdk_workspace_bytes(int32_t batch, int32_t num_q_heads, int32_t head_dim, int32_t num_splits);

/* Number of int32 counters fdk_decode can use for these arguments (see fdk_decode_args.counters). */
int64_t fdk_counters_len(const fdk_decode_args* args);

/* Split kernel then combine kernel; a single launch when the plan has one split (or with FDK_FLAG_SINGLE_LAUNCH). */
int fdk_decode(const fdk_decode_args* args, void* hip_stream);

/* fdk_decode without a workspace argument and without any allocation.  It has no counterpart in the reference;
 * it is for callers that cannot allocate device memory or call anything that might: code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  The split partials go to a scratch array of
 * FDK_STATIC_SCRATCH_BYTES that is part of the library's code object (one copy per GPU, held until the process
 * ends); args->workspace and args->counters are ignored (one workgroup per item, never the work-queue form; without
 * counters FDK_FLAG_SINGLE_LAUNCH has nothing to draw tickets on and the call runs as split kernel + combine kernel).
 * Same plan, same kernels and bit-identical results as fdk_decode with a caller-owned workspace.
 *   - A plan whose partials exceed the scratch is rejected with FDK_EWORKSPACE before anything is launched
 *     (fdk_workspace_bytes(batch, num_q_heads, head_dim, plan.num_splits) > FDK_STATIC_SCRATCH_BYTES).
 *   - All calls on one GPU share that GPU's scratch and its contents are unspecified between calls: two calls
 *     that overlap in time on one GPU (different streams, or graph replays running concurrently) race.
 *   - The first call on a device looks up the device address of the scratch (no allocation, but not a
 *     stream operation): make one call per device before capturing a graph. */
#define FDK_STATIC_SCRATCH_BYTES (32u << 20)
int fdk_decode_static(const fdk_decode_args* args, void* hip_stream);

/* A length-feedback block (fdk_decode_args.length_feedback): 4 zeroed int32 in pinned host memory that the current GPU
 * can write.  *host is where the CPU reads them, *device what goes into the argument block.  No counterpart in the
 * reference.  fdk_length_feedback_free takes the host pointer. */
int fdk_length_feedback_alloc(int32_t** host, int32_t** device);
int fdk_length_feedback_free(int32_t* host);

/* Split kernel only: fills the workspace with per-split (o, lse); args->out/lse unused. */
int fdk_decode_splitkv(const fdk_decode_args* args, void* hip_stream);

/* Combine kernel only: merges the workspace written by fdk_decode_splitkv with the same args. */
int fdk_combine(const fdk_decode_args* args, void* hip_stream);

/* Merge R per-rank local results into the global attention output. */
int fdk_combine_ranks(const fdk_combine_ranks_args* args, void* hip_stream);

/* 16-bit rows to MXFP4 rows and back (see fdk_mxfp4_args). */
int fdk_mx_quantize(const fdk_mxfp4_args* args, void* hip_stream);
int fdk_mx_dequantize(const fdk_mxfp4_args* args, void* hip_stream);

/* Normalise, rotate and append the new tokens (see fdk_kv_append_args). */
int fdk_kv_append(const fdk_kv_append_args* args, void* hip_stream);

/* ... with explicit positions, or into an MXFP4 cache (see fdk_kv_append_axes_args). */
int fdk_kv_append_axes(const fdk_kv_append_axes_args* args, void* hip_stream);

/* Add the attention weights of one query token per sequence to the cached tokens' sums (see fdk_attn_weights_args). */
int fdk_accumulate_weights(const fdk_attn_weights_args* args, void* hip_stream);

/* Evict the tokens of least weight (see fdk_kv_evict_args).  Calls that overlap in time need distinct workspaces. */
int fdk_kv_evict(const fdk_kv_evict_args* args, void* hip_stream);
size_t fdk_kv_evict_workspace_bytes(const fdk_kv_evict_args* args); /* (reads sizes only; for the current device) */

#ifdef __cplusplus
}
#endif
#endif /* FDK_H_ */
