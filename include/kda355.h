/*
 * kda355.h -- C ABI of the MI355X (gfx950) KDA library libkda355.so.
 *
 * KDA (Kimi Delta Attention): the gated delta rule with a per-key-channel decay, head dim K = V = 128, fp32
 * state stored V-major [V][K] (128 x 128 floats = 64 KiB per (sequence, head)).
 *
 * Every entry point takes a POD argument struct of raw device pointers, element strides and sizes plus a
 * hipStream_t, launches asynchronously on that stream and returns a status code.  Nothing here allocates device
 * memory, synchronizes, or keeps per-call global state, so every launch entry point is safe inside HIP-graph
 * capture and re-entrant across threads and streams.  bf16 / fp16 tensors are passed as `const void*`.
 * The stream has to be one of the current device (hipSetDevice; stream 0 always is), and all pointers that device's.
 *
 * Status codes: 0 = launched; KDA355_EINVAL (-1) = invalid arguments (nothing launched, kda355_last_error()
 * names the argument); KDA355_ELAUNCH (-2) = the HIP launch failed.
 *
 * Which reference interface each entry point replaces (caoshiyi/eat-kernels paths):
 *   kda355_recurrent_launch       vLLM fused_recurrent_kda as called by the Kimi layer
 *                                 (kda/mi350x/benchmark/vllm_reference/kda.py:488-502, 560-575) and the recurrent
 *                                 core of the decode kernel's `run` binding (kda/mi350x/kda/decode/kda_v14_b.cu:
 *                                 3266-3312, slot rules `slots()` :1013-1042)
 *   kda355_decode_launch          the fused decode / spec-verify step of the vLLM-ROCm Kimi layer, `decode(mixed_qkv,
 *                                 conv_state, ...)` (kda/mi350x/kda/kernel.py:212-216; semantics
 *                                 kda/mi350x/reference.py:104-181; input contract kda/mi350x/kda/decode/kernel_v13_a.py:
 *                                 697-735; slot rules kda/mi350x/kda/decode/kda_v14_b.cu:1013-1042)
 *   kda355_spec_commit_launch     the commit of an accepted draft length (kda/mi350x/reference.py:117-121 reads the
 *                                 state after token a-1; this copies it to the sequence's pool slot)
 *   kda355_prefill_plan           kda_build_meta (kda/mi350x/kda/prefill/kernel.h:100-102) and prepare_prod
 *                                 (kda/mi350x/kda/prefill/main.cpp:103-130): host-only schedule tables
 *   kda355_prefill_workspace_bytes  kda_workspace_floats (kda/mi350x/kda/prefill/kernel.h:90-91)
 *   kda355_prefill_launch         kda_prefill_kernel_launch (kda/mi350x/kda/prefill/kernel.h:33-56) with the
 *                                 KdaPool production contract (kernel.h:19-31)
 */
#ifndef KDA355_H
#define KDA355_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* kda355_stream_t; /* == hipStream_t */

#define KDA355_EINVAL (-1)
#define KDA355_ELAUNCH (-2)
#define KDA355_HEAD_DIM 128
#define KDA355_CHUNK 64
/* Smallest per-token log-decay the chunked prefill uses: its diagonal Gram blocks hold e^{+-8 g} over 8 tokens, which
   for g >= -9 stays inside 2^{+-104}, where fp32 and bf16 are normal with room for the low half of a bf16 pair (the
   MFMAs flush subnormal operands).  A log-decay below it (given, or formed in the kernel from a lower_bound below it)
   is raised to it, which changes the state by less than e^{-9} = 1.2e-4 of the affected channel.  The
   reference guards the same range by recomputing overflowed slices in fp32 (kda/mi350x/kda/kernel.py:113-128). */
#define KDA355_MIN_LOG_DECAY (-9.0f)

/* ------------------------------------------------------------------------------------------------ recurrent */

/* flags of KdaRecurrentArgs */
#define KDA355_REC_NORMALIZE_QK 1u  /* q, k <- x * rsqrt(sum x^2 + 1e-6) in the kernel (kda/mi350x/reference.py:159-160) */
#define KDA355_REC_RAW_GATE 2u      /* g is bf16 raw_g: g = lower_bound * sigmoid(exp(A_log[h]) * (raw_g + dt_bias[h,k])) */
#define KDA355_REC_RAW_BETA 4u      /* beta is bf16 raw_beta: beta = sigmoid(raw_beta) */
#define KDA355_REC_PER_TOKEN 8u     /* write the state after every token t to write_idx[n, t] (spec verify);
                                       otherwise the final state goes back to the read row (plain decode) */
#define KDA355_REC_SLOT0_RESERVED 16u /* row 0 of read_pool is the padding slot: never read, never written */
#define KDA355_REC_WRITE_SLOT0_RESERVED 32u /* the same rule for write_pool (PER_TOKEN destinations) */

/*
 * Recurrent decode / speculative verify over B sequences x S tokens (T = B*S rows, row n*S + t is token t of
 * sequence n), H heads.  Per (n, h):
 *     read row   r = read_idx[n * read_idx_stride + (num_accepted ? clamp(num_accepted[n], 1, S) - 1 : 0)]
 *     S0         = read_pool[r]      (a padding row -- outside [0, read_slots), or 0 with SLOT0_RESERVED -- is
 *                                     never read; the sequence is skipped and its output rows are zero)
 *     per token: S *= exp(g_t) (key axis);  u = beta_t (v_t - S k_t);  S += u k_t^T;  o_t = scale * S q_t
 *     writes     PER_TOKEN: write_pool[write_idx[n*S + t]] = state after token t (padding rows skipped);
 *                otherwise read_pool[r] = final state.
 * The reference's spec-verify mapping (kda/mi350x/reference.py:135-143,168-171) is read_pool == write_pool,
 * read_idx == write_idx == state_indices [B, S], read_idx_stride = S, num_accepted given, PER_TOKEN.
 */
typedef struct KdaRecurrentArgs {
    const void* q;              /* bf16 [T, H, 128], row stride qkv_row_stride elements */
    const void* k;
    const void* v;
    const void* g;              /* fp32 [T, H, 128] log-decay, or bf16 raw_g with RAW_GATE; row stride g_row_stride */
    const void* beta;           /* fp32 [T, H] activated, or bf16 raw_beta with RAW_BETA; row stride beta_row_stride */
    const float* A_log;         /* [H]        (RAW_GATE only) */
    const float* dt_bias;       /* [H * 128]  (RAW_GATE only) */
    float* read_pool;           /* [read_slots, H, 128, 128] fp32 V-major, slot stride read_slot_stride floats */
    float* write_pool;          /* PER_TOKEN destination pool (may equal read_pool) */
    const int32_t* read_idx;    /* [B, read_idx_stride] */
    const int32_t* num_accepted;/* [B] or NULL */
    const int32_t* write_idx;   /* [B, S] (PER_TOKEN) or NULL */
    void* out;                  /* bf16 [T, H, 128], row stride out_row_stride elements */
    int64_t qkv_row_stride, g_row_stride, beta_row_stride, out_row_stride;
    int64_t read_slot_stride, read_slots, write_slot_stride, write_slots;
    int32_t B, S, H, read_idx_stride;
    float scale, lower_bound;
    uint32_t flags;
    int32_t reserved;
} KdaRecurrentArgs;

int kda355_recurrent_launch(const KdaRecurrentArgs* args, kda355_stream_t stream);

/*
 * Commit of an accepted draft length: for each sequence n with a = clamp(num_accepted[n], 1, S),
 * pool[pool_idx[n]] = scratch[scratch_idx[n*S + a - 1]] (all H heads; padding rows skipped as above).
 */
typedef struct KdaSpecCommitArgs {
    const float* scratch;       /* [scratch_slots, H, 128, 128] */
    float* pool;                /* [pool_slots, H, 128, 128] */
    const int32_t* scratch_idx; /* [B, S] */
    const int32_t* pool_idx;    /* [B] */
    const int32_t* num_accepted;/* [B] */
    int64_t scratch_slot_stride, scratch_slots, pool_slot_stride, pool_slots;
    int32_t B, S, H;
    uint32_t flags;             /* KDA355_REC_SLOT0_RESERVED applies to the pool (scratch rows may use 0) */
} KdaSpecCommitArgs;

int kda355_spec_commit_launch(const KdaSpecCommitArgs* args, kda355_stream_t stream);

/* ------------------------------------------------------------------------------------------------ fused decode */

/*
 * Fused decode / speculative verify of B sequences x S tokens (T = B*S rows, row n*S + t is token t of sequence n),
 * H heads, dim = H * 128, per (n, h) and token t:
 *     conv      x = SiLU(sum_j window[t + j] * conv_weight[:, j]) over the head's q | k | v channels, where window =
 *               3 history taps of conv_state[cs] followed by the S rows of mixed_qkv (width-4 causal depthwise conv)
 *     q, k      x * rsqrt(sum x^2 + 1e-6);  q *= 128^-1/2
 *     gate      g = lower_bound * sigmoid(exp(A_log[h]) * (gate + dt_bias));  beta = sigmoid(beta)
 *     rule      S *= exp(g) (key axis);  u = beta (v - S k);  S += u k^T;  o = S q
 *     output    y = bf16(o) * rsqrt(mean(bf16(o)^2) + norm_eps) * norm_weight * sigmoid(out_gate)   (bf16)
 * plain decode (num_accepted == NULL, state_indices [B]): rd = cs = state_indices[n]; the final state goes back to
 *     ssm_state[rd]; conv_state[cs] taps [0, 3) <- the last 3 window rows (taps beyond 3 are untouched).
 * spec verify (num_accepted [B], state_indices [B, S]): a = clamp(num_accepted[n], 1, S), rd = state_indices[n, a-1],
 *     cs = state_indices[n, 0]; history taps [a-1, a+2); the state after token t goes to ssm_state[state_indices[n, t]]
 *     (rows <= 0 skipped); conv_state[cs] taps [0, 2 + S) <- window rows [1, 3 + S).
 * Rows <= 0 or outside the pool are padding: a sequence whose rd or cs is padding gets zero output rows and writes
 * nothing.  The vLLM page layout (conv_state and ssm_state as strided views into one byte pool) is expressed by the
 * slot strides.  S <= 16.
 */
typedef struct KdaDecodeArgs {
    const void* mixed_qkv;      /* bf16 [T, 3 * dim], row stride mixed_row_stride elements (16-byte aligned rows) */
    void* conv_state;           /* bf16 [conv_slots, conv_taps, 3 * dim]: slot / tap strides in elements */
    const float* conv_weight;   /* [3, 4, dim] dense: (q | k | v, tap, channel) */
    const void* gate;           /* bf16 [T, H, 128], row stride gate_row_stride elements */
    const void* beta;           /* bf16 [T, H] logits, row stride beta_row_stride */
    const void* out_gate;       /* bf16 [T, dim], row stride out_gate_row_stride */
    const float* A_log;         /* [H] */
    const float* dt_bias;       /* [dim] */
    const float* norm_weight;   /* [128] */
    float* ssm_state;           /* [ssm_slots, H, 128, 128] fp32 V-major, slot stride ssm_slot_stride floats */
    const int32_t* state_indices;  /* [B] (plain) or [B, S] (spec), dense */
    const int32_t* num_accepted;   /* [B] or NULL (plain decode) */
    void* out;                  /* bf16 [T, dim], row stride out_row_stride */
    int64_t mixed_row_stride, gate_row_stride, beta_row_stride, out_gate_row_stride, out_row_stride;
    int64_t conv_slot_stride, conv_tap_stride, conv_slots, ssm_slot_stride, ssm_slots;
    int32_t B, S, H, conv_taps;
    float norm_eps, lower_bound;
    uint32_t flags;             /* 0 */
    int32_t reserved;
    void* workspace;            /* NULL, or KDA355_DECODE_WS_BYTES of device memory whose first 256 bytes (the
                                   counters) are zero before the first launch: launches of at most 64 (sequence, head)
                                   pairs (B * H) then split each state over 4 workgroups, the last of which finishes the
                                   head's outputs.  Each such launch leaves the counters zero again (the rest is
                                   written before it is read); launches that may run at the same time on one GPU need
                                   workspaces of their own.  No counterpart in the reference's decode entry (its
                                   single-launch small-batch kernel is kda/mi350x/kda/decode/kda_v14_b.cu:1856-). */
} KdaDecodeArgs;

/* Bytes of the decode workspace: 64 int32 counters, then 64 x 4 x 16 fp32 partial sums of squares. */
#define KDA355_DECODE_WS_BYTES 16640

int kda355_decode_launch(const KdaDecodeArgs* args, kda355_stream_t stream);

/* ------------------------------------------------------------------------------------------------ prefill */

/* flags of KdaPrefillPlanIn / KdaPrefillArgs */
#define KDA355_PF_NORMALIZE_QK 1u  /* q, k <- x / max(|x|, 1e-6) in the kernel (kda/mi350x/reference.py:59-60) */
#define KDA355_PF_RAW_GATE 2u      /* g is bf16 raw_g: g = lower_bound * sigmoid(exp(A_log[h]) * (raw_g + dt_bias[h,k])) */
#define KDA355_PF_RAW_BETA 4u      /* beta is bf16 raw_beta (any row stride): beta = sigmoid(raw_beta) */
#define KDA355_PF_POOL 8u          /* states live in a paged pool: read state_pool[state_idx[n]] when has_initial_state[n]
                                      (else start from zero and never read the row), write the final state there */
#define KDA355_PF_CK_SINGLE 16u    /* one checkpoint per sequence: the state after ck_offsets[n] tokens (a positive
                                      multiple of 64, <= the length; planned on the host) goes to ck_pool[ck_idx[n]]
                                      when ck_idx[n] >= 0 (kda/mi350x/reference.py:38-41,52-57) */
#define KDA355_PF_CK_EVERY 32u     /* every-n checkpoints: row j of sequence n (j < ceil(len_n / ck_every)) is the state
                                      before token j * ck_every, stored to ck_pool[ck_idx[row_start_n + j]] with
                                      row_start_n = sum of the earlier sequences' row counts (kda/b200/kda_b200.py:19-22) */
#define KDA355_PF_PRECISE 64u      /* the solve's and the state update's fp16 operands as fp16 pairs (22 bits): about half
                                      the state error on chunks of nearly parallel keys with beta ~ 1, 3-17 % more time.
                                      No counterpart in the reference (its prefill precision is fixed). */
#define KDA355_PF_CHUNK64 128u     /* keep the 64-token kernel (and the plan's workgroup lists) where the plan chose the
                                      32-token kernel (KdaPrefillPlan.chunk32); a comparison and test switch.  No
                                      counterpart in the reference. */

/* Host-side plan input: the layout only (never the data). */
typedef struct KdaPrefillPlanIn {
    const int64_t* cu_seqlens;  /* host [N + 1] token offsets */
    const int32_t* ck_offsets;  /* host [N] single-checkpoint offsets (tokens) or NULL */
    int32_t N, H;
    int32_t ck_every;           /* every-n interval in tokens (multiple of 64) or 0 */
    int32_t num_cus;            /* CUs of the device (0: 256); long sequences are split into pieces of >= 16 chunks
                                   when that shortens the schedule (the chains alone would leave CUs idle, or the
                                   longest ones would finish well after the rest) */
    uint32_t flags;             /* unused (0): checkpoint work is scheduled for every kind the layout defines */
    int32_t reserved;
} KdaPrefillPlanIn;

/* Filled by kda355_prefill_plan. */
typedef struct KdaPrefillPlan {
    int64_t T;
    int32_t N, H, num_chunks, num_chains, max_chain_chunks, ck_every;
    int64_t table_words;        /* int32 words of the schedule table (copy it to the device once per layout) */
    int64_t workspace_bytes;    /* device workspace the launch needs (256-byte aligned) */
    int64_t ck_rows;            /* every-n rows the layout writes (sum over n of ceil(len_n / ck_every)) */
    uint32_t magic, flags;
    int32_t num_pieces;         /* pieces of split sequences (0: no sequence is split) */
    int32_t num_split;          /* split sequences */
    int32_t num_fix_tasks;      /* groups of <= 2 chunks of the later pieces of split sequences (outputs completed after
                                   the scan) */
    int32_t num_ck_tasks;       /* checkpoints inside later pieces (composed after the scan) */
    int32_t chunk_grid;         /* workgroups of the chunk launch: 0 = one per (chain, head); > 0 (layouts without
                                   split sequences whose (chain, head) pairs outnumber the CUs) = that many
                                   workgroups, each walking a list of (chain, head) pairs in turn */
    int32_t chunk32;            /* 1: the launch runs the 32-token chunk kernel, one workgroup per (chain, head) and two
                                   per CU (layouts without split sequences whose items outnumber the CUs, when its
                                   simulated schedule beats chunk_grid's); launches with KDA355_PF_PRECISE or
                                   KDA355_PF_CHUNK64 keep the 64-token kernel.  May be set to 1 by the caller for any
                                   plan without split sequences. */
} KdaPrefillPlan;

/*
 * Schedule of one batch layout (host only, no device call).  Call once with tables == NULL to get
 * plan->table_words, then with a host buffer of that many int32 words, and copy the buffer to the device.
 */
int kda355_prefill_plan(const KdaPrefillPlanIn* in, KdaPrefillPlan* plan, int32_t* tables, int64_t capacity);
int64_t kda355_prefill_workspace_bytes(const KdaPrefillPlan* plan);

/*
 * Chunked prefill over a packed varlen batch (T tokens, N sequences, H heads):
 *   q, k, v [T, H, 128] bf16; g [T, H, 128] fp32 log-decay or bf16 raw gate; beta [T, H] fp32 or bf16 raw;
 *   out [T, H, 128] bf16.  Per (n, h) the token recurrence of kda/mi350x/reference.py:85-91 with scale.
 * States: KDA355_PF_POOL -> state_pool [state_slots, H, 128, 128] (rows dense, slot stride state_slot_stride floats),
 * else initial_state [N, H, 128, 128] (NULL = zeros) and final_state [N, H, 128, 128], contiguous.
 * Checkpoint rows go to ck_pool (fp32, or bf16 rounded to nearest even when ck_dtype == 1), slot stride in elements.
 * Rows outside [0, slots) are skipped.  Asynchronous on `stream`; no host synchronization.
 */
typedef struct KdaPrefillArgs {
    const void* q;
    const void* k;
    const void* v;
    const void* g;
    const void* beta;
    const float* A_log;
    const float* dt_bias;
    void* out;
    float* state_pool;
    const int32_t* state_idx;        /* [N] */
    const uint8_t* has_initial_state;/* [N] bool */
    const float* initial_state;
    float* final_state;
    void* ck_pool;
    const int32_t* ck_idx;           /* CK_SINGLE: [N] rows; CK_EVERY: [ck_rows] rows */
    const int32_t* tables;           /* device copy of the plan's schedule table */
    void* workspace;                 /* >= plan->workspace_bytes, 256-byte aligned */
    int64_t qkv_row_stride, g_row_stride, beta_row_stride, out_row_stride;  /* elements between tokens, each
                                                                              in [0, 2^21) */
    int64_t state_slot_stride, state_slots, ck_slot_stride, ck_slots;
    int64_t T;
    int32_t N, H;
    float scale, lower_bound;
    uint32_t flags;
    int32_t ck_dtype;                /* 0 fp32, 1 bf16 */
    const KdaPrefillPlan* plan;
} KdaPrefillArgs;

int kda355_prefill_launch(const KdaPrefillArgs* args, kda355_stream_t stream);

/*
 * kda355_prefill_launch without a caller workspace.  No counterpart in the reference: it is for callers that cannot
 * allocate device memory (code under graph capture with no allocator at hand, tight serving loops, harnesses that
 * forbid allocation).  args->workspace must be NULL; the workspace of split layouts comes from a static device array
 * of KDA355_NOALLOC_SCRATCH_BYTES that every GPU the library runs on holds until the process ends, and a plan whose
 * workspace_bytes exceeds it is rejected with KDA355_EINVAL (config-2-sized layouts need ~1 GB: use
 * kda355_prefill_launch there).  The call allocates nothing.  Calls that overlap on one GPU share the array and
 * race: serialize them (one stream).  Nothing in the array has to start at zero.
 */
#define KDA355_NOALLOC_SCRATCH_BYTES (256ull << 20)
int kda355_prefill_launch_noalloc(const KdaPrefillArgs* args, kda355_stream_t stream);

/* ------------------------------------------------------------------------------------------------ latent attention */

/*
 * The attention layers between the KDA layers of a hybrid model: every token leaves one latent vector of 512 values and
 * a positional part of 64 (rotated or not, as the model has it) that all heads share.  Head dims: 128 + 64 for q and k,
 * 128 for v.  No counterpart in the reference, which holds KDA layers only.
 *
 * Cache: [pages, page_size, 576] in 16-bit elements, the token rows (latent | positional part) dense within a page, any
 * page stride.  Page numbers outside [0, pages) are holes: their tokens are never read and take no part.
 *
 * A cache in 4 bits: [pages, page_size, 400] bytes.  A row is 256 bytes of codes (value 2 i in the low half of byte i), 16 scale
 * bytes of 32 consecutive values each, and the positional part in 16 bits.  A code is a sign (8) and one of 0, 0.5, 1, 1.5, 2, 3,
 * 4, 6; a scale byte b stands for 2^(b - 127), 255 for NaN (a NaN group).  Readers round code x scale to their 16-bit type: with
 * what kda355_latent4_append_launch writes for that type the products are numbers of it.
 */
#define KDA355_LATENT_DIM 512
#define KDA355_LATENT_PE 64
#define KDA355_LATENT_ROW 576
#define KDA355_LATENT_ROW_4BIT 400
#define KDA355_LATENT_GROUP 32
#define KDA355_DTYPE_BF16 0
#define KDA355_DTYPE_FP16 1
#define KDA355_LATENT_CAUSAL 1u

/*
 * Expanded form over N packed sequences: sequence n has queries [cu_q[n], cu_q[n + 1]) and keys [cu_k[n], cu_k[n + 1]).
 * With its lengths Lq and Lk and KDA355_LATENT_CAUSAL, query i sees keys j <= i + Lk - Lq (the queries are the last
 * tokens); without, all of them.  z = scale (q[:128] . k + q[128:] . k_pe);  out = softmax(z) v;  lse = log sum e^z.  A
 * query that sees no key gets zeros and an lse of -inf.  Keys that a query does not see never reach its output, whatever
 * they hold.  Rows of no sequence are not written.  Sums and softmax statistics are fp32; weights are rounded to the type for
 * their product with the values.  Scores z have to stay within +-2^24.
 */
typedef struct KdaLatentPrefillArgs {
    const void* q;       /* [Tq, H, 192], strides in elements */
    const void* k;       /* [Tk, H, 128] */
    const void* v;       /* [Tk, H, 128] */
    const void* k_pe;    /* [Tk, 64] */
    void* out;           /* [Tq, H, 128] */
    float* lse;          /* [Tq, H] dense, natural logarithm, or NULL */
    const int32_t* cu_q; /* [N + 1] on the device, not decreasing, within [0, Tq] (clamped to it) */
    const int32_t* cu_k; /* [N + 1], the same for Tk */
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, pe_row, out_row, out_head;
    int64_t Tq, Tk;
    void* workspace;     /* kda355_latent_prefill_workspace_bytes(args), 256-byte aligned; nothing in it has to start at
                            zero, launches that may overlap need their own */
    int64_t workspace_bytes;
    int32_t N, H, dtype;
    uint32_t flags;      /* KDA355_LATENT_CAUSAL or 0 */
    float scale;         /* positive */
    int32_t num_cus;     /* CUs to fill (0: 256) */
} KdaLatentPrefillArgs;

/* Bytes of workspace for these sizes (pointers and strides are not looked at), or KDA355_EINVAL.  Room for every cut of the
   keys that the lengths on the device may ask for: 66560 bytes for each of up to 8 num_cus parts of 128 rows, 136 MB with 256
   CUs however long the prompt (less where few rows and keys cannot be cut so far: 0.5 MB for 100 rows of 4 heads over 300 keys). */
int64_t kda355_latent_prefill_workspace_bytes(const KdaLatentPrefillArgs* args);
int kda355_latent_prefill_launch(const KdaLatentPrefillArgs* args, kda355_stream_t stream);

/*
 * Absorbed form over the paged cache, B sequences x S tokens (row n * S + s is token s of sequence n): with c_j the latent
 * and r_j the positional part of cached token j, z = scale (q_latent . c_j + q_pe . r_j);  out = sum softmax(z) c_j.
 * seq_lens[n] cached tokens, the S new ones among them: token s sees j < seq_lens[n] - (S - 1 - s).  seq_lens is clamped
 * to [0, table_width * page_size].
 * With prefix_table, every sequence first sees the prefix_len[0] tokens of those pages (all S tokens see all of them),
 * then its own; the prefix is read once for all rows.  A row that sees nothing gets zeros and an lse of -inf.  scale must be
 * positive, B * S * H below 2^29.  Precision and range of the scores as above.
 */
typedef struct KdaLatentDecodeArgs {
    const void* q_latent;        /* [B * S, H, 512], strides in elements */
    const void* q_pe;            /* [B * S, H, 64] */
    const void* cache;           /* [pages, page_size, 576] */
    const int32_t* block_table;  /* [B, table_width], row stride table_stride */
    const int32_t* seq_lens;     /* [B] */
    const int32_t* prefix_table; /* [prefix_width] or NULL */
    const int32_t* prefix_len;   /* [1] (with prefix_table) */
    void* out;                   /* [B * S, H, 512] */
    float* lse;                  /* [B * S, H] dense, or NULL */
    void* workspace;             /* kda355_latent_decode_workspace_bytes(args), 256-byte aligned; nothing in it has to
                                    start at zero, launches that may overlap need their own */
    int64_t ql_row, ql_head, qp_row, qp_head, out_row, out_head;
    int64_t page_stride, pages, table_stride, workspace_bytes;
    int32_t B, S, H, page_size, table_width, prefix_width;
    int32_t dtype, num_cus;      /* num_cus: workgroups the launch fills (0: 256) */
    float scale;
    uint32_t flags;              /* 0 */
} KdaLatentDecodeArgs;

/* Bytes of workspace for these sizes (pointers and strides are not looked at), or KDA355_EINVAL.  65792 bytes for 32 rows of a
   part: num_cus parts and one for each group of up to 64 rows of a sequence, and num_cus more with a prefix.  With 256 CUs 17 MB
   for one sequence of 12 heads, 42 MB for 64 of 64 heads, 303 MB for 128 x 8 tokens of 128 heads, 842 MB for 512 x 8 of 96. */
int64_t kda355_latent_decode_workspace_bytes(const KdaLatentDecodeArgs* args);
int kda355_latent_decode_launch(const KdaLatentDecodeArgs* args, kda355_stream_t stream);
/* The same over a cache in 4 bits: page_stride is in bytes, everything else (the workspace too) as above. */
int kda355_latent4_decode_launch(const KdaLatentDecodeArgs* args, kda355_stream_t stream);

/*
 * What the cached tokens were given by an attention step of the absorbed form: weights[n, j] += sum over the S * H rows of
 * sequence n that see token j of e^(z - lse[row]), z as above.  lse is what the step left (NULL is refused): with a shared prefix
 * its weights count in lse, and only the sequence's own tokens are written.  Rows with an lse of -inf give nothing, tokens in holes
 * get nothing, weights past the tokens stay as they are.  Sums are fp32, in an order that the sizes alone decide.
 */
typedef struct KdaLatentWeightsArgs {
    const void* q_latent;        /* [B * S, H, 512], strides in elements */
    const void* q_pe;            /* [B * S, H, 64] */
    const void* cache;           /* [pages, page_size, 576] in 16 bits or [pages, page_size, 400] bytes */
    const int32_t* block_table;  /* [B, table_width], row stride table_stride */
    const int32_t* seq_lens;     /* [B], clamped to [0, table_width * page_size] */
    const float* lse;            /* [B * S, H] dense */
    float* weights;              /* [B, table_width * page_size], row stride weights_row */
    int64_t ql_row, ql_head, qp_row, qp_head, weights_row;
    int64_t page_stride, pages, table_stride;  /* page_stride: 16-bit elements, bytes of a cache in 4 bits */
    int32_t B, S, H, page_size, table_width, dtype;
    int32_t cache_bits;          /* 16 or 4 */
    int32_t num_cus;             /* CUs to fill (0: 256) */
    float scale;                 /* positive */
    uint32_t flags;              /* 0 */
} KdaLatentWeightsArgs;

int kda355_latent_weights_launch(const KdaLatentWeightsArgs* args, kda355_stream_t stream);

/*
 * Token rows into pages and back.  append: cache row slots[t] (page * page_size + offset) <- latent[t] | k_pe[t]; slots
 * outside [0, pages * page_size) are skipped, those inside have to differ (of two tokens of one slot pieces of both may stay).  gather: out[cu[n] + j] <- token
 * j of sequence n, for j < cu[n + 1] - cu[n]; tokens of holes or past the table give zero rows.
 */
typedef struct KdaLatentTokensArgs {
    const void* latent;          /* append: [T, 512] */
    const void* k_pe;            /* append: [T, 64] */
    void* cache;                 /* [pages, page_size, 576] */
    const int64_t* slots;        /* append: [T] */
    const int32_t* block_table;  /* gather: [N, table_width] */
    const int32_t* cu;           /* gather: [N + 1] on the device, not decreasing; rows outside [0, T) are skipped */
    void* out;                   /* gather: [T, 576], row stride out_row */
    int64_t latent_row, pe_row, out_row, page_stride, pages, table_stride, T;
    int32_t page_size, table_width, N;
    int32_t dtype;               /* of latent, k_pe and out; looked at for caches in 4 bits only */
} KdaLatentTokensArgs;

int kda355_latent_append_launch(const KdaLatentTokensArgs* args, kda355_stream_t stream);
int kda355_latent_gather_launch(const KdaLatentTokensArgs* args, kda355_stream_t stream);
/*
 * The same with a cache in 4 bits (page_stride in bytes).  append: with a the largest |x| of 32 values, the scale is 2^e,
 * e = floor(log2 a) - 2, and 1 more where a > 7 x 2^e, in [-125, 125] (bf16) or [-23, 13] (fp16); a value becomes the nearest
 * code x 2^e, ties to the even code, at most 6 x 2^e, and is off by at most a / 5; by a / 4 where the upper limit holds e down (a > 57344 in
 * fp16, 7 x 2^125 in bf16: the largest value reads back as 6 x 2^e), and by 2^-127 if that is more where bf16's lower limit holds it up (a <
 * 2^-123).  A group with an infinite value or a NaN reads as NaN throughout.
 */
int kda355_latent4_append_launch(const KdaLatentTokensArgs* args, kda355_stream_t stream);
int kda355_latent4_gather_launch(const KdaLatentTokensArgs* args, kda355_stream_t stream);

/* ------------------------------------------------------------------------------------------------ pages of a cache */

/*
 * Page bookkeeping on the device: sequences are rows of block_table (entries outside [0, pages) are holes), a page holds
 * page_size tokens and ref_counts[page] sequences hold it.  free_pages[0 .. num_free[0]) is a stack of the pages nobody
 * holds, the next one at its top; entries past it are -1.  Nothing is read back to the host, so the calls can be captured;
 * results do not depend on timing.  No counterpart in the reference (its caller manages slots on the host).
 *
 * A pool is one layer's tensor [slots, ...] with dense rows of row_bytes (a multiple of 16) at 16-byte aligned addresses.
 */
#define KDA355_MAX_POOLS 24
typedef struct KdaPool {
    void* base;
    int64_t row_bytes, slot_stride; /* bytes */
    int64_t slots;
} KdaPool;

typedef struct KdaPagesArgs {
    KdaPool pool[KDA355_MAX_POOLS];
    int32_t num_pools, n;        /* n: pairs / rows given */
    const int32_t* src;          /* copy: [n] rows;  fork: [n] parents;  free: [n] rows */
    const int32_t* dst;          /* copy: [n] rows;  fork: [n] children */
    int32_t* block_table;        /* [rows, table_width], row stride table_stride */
    int32_t* seq_lens;           /* [rows] */
    int32_t* ref_counts;         /* [pages] */
    int32_t* free_pages;         /* [pages] */
    int32_t* num_free;           /* [1] */
    int32_t* workspace;          /* fork: 2 n words;  compact: 2 pages + 2 words */
    int64_t table_stride;
    int32_t rows, table_width, pages, page_size;
} KdaPagesArgs;

/* pool[dst[i]] <- pool[src[i]] in every pool; pairs with a row outside a pool are skipped there.  No dst may be another
   pair's src or dst. */
int kda355_copy_rows_launch(const KdaPagesArgs* args, kda355_stream_t stream);
/* Sequence dst[i] becomes a copy of src[i], in the order of i: its full pages are shared, a part-filled last page is copied
   in every pool to a page taken from the stack.  Holes stay holes: a part-filled last page that is one takes no page.  Where
   the stack is empty, the child gets length 0 and no pages.  What the child row held before is overwritten, not released.
   Pairs outside [0, rows) are skipped; children must differ from one another and from every parent. */
int kda355_fork_pages_launch(const KdaPagesArgs* args, kda355_stream_t stream);
/* Sequences src[i] (all different) give up the pages of their seq_lens tokens; rows become holes, lengths 0.  Pages that
   nobody holds any more go onto the stack, the highest first.  Entries past the tokens become holes without being given up:
   where pages are reserved ahead, raise seq_lens to cover them first (holes among them are skipped). */
int kda355_free_pages_launch(const KdaPagesArgs* args, kda355_stream_t stream);
/* With L pages held: the i-th held page at or above L moves into the i-th free one below L, in every pool; tables, counts
   and the stack (pages - 1 down to L, so that L is taken next) follow.  Lists of pages kept elsewhere are not rewritten: keep
   the pages of a shared prefix as a row of block_table. */
int kda355_compact_pages_launch(const KdaPagesArgs* args, kda355_stream_t stream);

/*
 * Sequences src[i] cut to `keep` tokens in every layer.  Of a sequence of len > keep tokens stay: the `recent` last; the fixed ones, all
 * up to the end of its last page with a reference count above 1; and of the others (from there to len - recent) the
 * keep - recent - fixed with the largest weights of the layer (a NaN is larger than any number, -0 is 0, ties go to the lower index).  With left = keep -
 * recent, the i-th token below `left` that goes gives its place to the i-th token that stays at or above it, in both the cache
 * and the weights; the recent ones follow in order.  Weights of places keep .. len - 1 become 0.  Pages behind the first
 * ceil(keep / page_size) are given up, those that nobody holds any more go onto the stack, the highest first; table entries past
 * the tokens (pages reserved ahead) move down behind the kept ones.
 *
 * A sequence stays as it is where len <= keep, an entry of its tokens' pages is a hole, or fixed > keep - recent.  Rows outside
 * [0, rows) are skipped, a row that is given twice is taken once.  Results do not depend on timing.
 * At most 65535 rows in one call (2^20 - 1 where the table holds no more than keep tokens: nothing can be cut), 2^30 tokens a table row.
 */
typedef struct KdaEvictLayer {
    void* cache;                 /* [pages, page_size] tokens of token_bytes, dense within a page */
    int64_t token_bytes;         /* a multiple of 16 */
    int64_t page_stride;         /* bytes, a multiple of 16 */
    float* weights;              /* [rows, table_width * page_size] */
    int64_t weights_row;         /* elements */
} KdaEvictLayer;

typedef struct KdaEvictArgs {
    KdaEvictLayer layer[KDA355_MAX_POOLS];
    int32_t num_layers, n;       /* n: rows given */
    const int32_t* src;          /* [n] */
    int32_t* block_table;        /* books as above */
    int32_t* seq_lens;
    int32_t* ref_counts;
    int32_t* free_pages;
    int32_t* num_free;
    void* workspace;             /* kda355_evict_tokens_workspace_bytes(args), 16-byte aligned */
    int64_t workspace_bytes;
    int64_t table_stride;
    int32_t rows, table_width, pages, page_size;
    int32_t keep, recent;        /* keep >= 1, 0 <= recent <= keep */
    uint32_t flags;              /* KDA355_EVICT_MORE: more layers follow in another call, the books stay as they are */
    int32_t reserved;
} KdaEvictArgs;
#define KDA355_EVICT_MORE 1u

/* Bytes of workspace for these sizes (pointers and strides are not looked at), or KDA355_EINVAL for sizes that the launch refuses.  At most
   128 MiB of lists (8 bytes for each of min(keep - recent, table_width * page_size - keep) tokens of a layer; those of one sequence's layers
   where they are more), 25 KiB and 16 bytes a part of 8192 tokens for 1024 (sequence, layer)s where a table row spans more than
   recent + 16384 tokens, and the lengths, counts and pages of the recent tokens of all rows. */
int64_t kda355_evict_tokens_workspace_bytes(const KdaEvictArgs* args);
int kda355_evict_tokens_launch(const KdaEvictArgs* args, kda355_stream_t stream);

/* ------------------------------------------------------------------------------------------------ misc */

/* Human-readable reason of the last KDA355_EINVAL / KDA355_ELAUNCH on the calling thread ("" if none). */
const char* kda355_last_error(void);
/* Library version (major * 10000 + minor * 100 + patch). */
int kda355_version(void);

#ifdef __cplusplus
}
#endif

#endif /* KDA355_H */
