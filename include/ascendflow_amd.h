/*
 * ascendflow_amd C ABI: MI355X (gfx950) sparse-MLA and flash-attention launchers.
 *
 * Drop-in counterparts of the launchers the reference's back end emits for its
 * three attention operators (src/backend/structured.py:573-649):
 *   int launch_<k>(void* stream, void* arg_<tensor>..., [void* workspace], [int64 sizes]);
 *   int kernel_config_<k>(int64_t cfg[5]);
 *   const char* kernel_metadata_<k>(void);
 *   int workspace_size_<k>(uint64_t* bytes, ...);   (src/backend/workspace.py:100-130)
 *
 * The reference specialises every size as a DSL constexpr; here the sizes are
 * runtime fields of a small parameter struct passed by pointer, because the
 * drop-in surface is the Python entry signature, not the Ascend binary.
 *
 * Conventions (all entry points):
 *  - every tensor argument is a device pointer to contiguous row-major memory;
 *    the caller allocates all tensors, outputs included, and keeps them
 *    pairwise disjoint (docs/guide/runtime.md:86-89 in the reference);
 *  - launches are asynchronous on `stream` (a hipStream_t, NULL = default);
 *  - return value: 0 on success, a negative AFA_E* code for a rejected
 *    configuration, or a positive hipError_t if the launch itself failed.
 *    Nothing is retried (src/runtime/kernel.py:59-63).
 */
#ifndef ASCENDFLOW_AMD_H
#define ASCENDFLOW_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  AFA_OK = 0,
  AFA_E_NULL = -1,        /* a required pointer is NULL */
  AFA_E_SHAPE = -2,       /* unsupported or inconsistent size */
  AFA_E_DTYPE = -3,       /* unsupported storage dtype */
  AFA_E_WORKSPACE = -4,   /* workspace missing or too small */
};

enum { AFA_DTYPE_BF16 = 0, AFA_DTYPE_F16 = 1 };

/* 8-bit codes of a quantised cache. */
enum { AFA_CODE_E4M3 = 0, AFA_CODE_INT8 = 1 };

/* Sizes and policy of one sparse_mla call
 * (examples/sparse_attention/attention.py:225-245). */
typedef struct SparseMlaParams {
  int32_t B, T, H, D;
  int32_t PAGE, RATIO, MAX_SEQ;
  int32_t ORI_BLOCKS, CMP_BLOCKS;
  int32_t WINDOW, TOPK, S, BM;
  int32_t dtype;            /* AFA_DTYPE_* of q, caches and attention_out */
  float scale;              /* SCALE, > 0 */
  /* Parts each (token, BM-head tile) key is split into, with a workspace: 0 =
   * automatic (after at most one full round of keys over 256 compute units,
   * the keys of the incomplete last round, into the number of parts a cost
   * model of the GPU finds cheapest, if any: decode with few requests), 1 =
   * never, 2..8 = every key. Parts run on different workgroups and store their
   * output normalised by their own denominator, with their running max and
   * denominator; a merge kernel combines them in part order, so results are
   * deterministic for a given value. No counterpart in the reference, whose
   * sizes are compile-time constants. */
  int32_t parts;
  /* KV ring of the persistent kernel (the plan path): 0 = automatic, 3 or 4
   * tiles of 32 rows. Three tiles keep one chunk in flight, four keep two.
   * Automatic takes four when ori_kv and cmp_kv together exceed MI355X's
   * 256 MiB Infinity Cache (rows then mostly come from HBM), else three; four
   * tiles are used only where the row-list ring fits next to them in LDS
   * (otherwise three). Results are bit-identical either way. No counterpart
   * in the reference. */
  int32_t ring;
  /* Optional debug image of the row selection, NULL normally: int32 [T, S, 2].
   * Entry r < n of token t is the r-th row of the compacted row list the
   * attention kernel streams for t (the LDS list it attends over, copied out
   * after it is built), as (cache, physical_row), cache 0 = ori_kv,
   * 1 = cmp_kv, in slot order (window positions, then compressed ranks,
   * duplicates kept); entries from n on are (-1, -1). A call with it set
   * resolves rows inside the attention kernel and splits no key. The
   * per-slot layout of the reference's gather workspace is
   * launch_sparse_mla_gather's. */
  int32_t* debug_rows;
  /* Optional f32 [T, H] output, NULL normally: the natural-log softmax
   * normaliser ln(sum_j e^(s_j) + e^sink[h]) of each (token, head), s_j =
   * SCALE * q.k_j over the selected rows (the sink alone for an empty
   * selection), i.e. the denominator of attention_out. The counterpart of the
   * softmax_lse output of the vendor operator the reference benchmarks against
   * (aclnnSparseFlashMla, benchmarks/references/sparse_mla_aclnn.py:100-130),
   * which the DSL kernel itself does not produce. */
  float* softmax_lse;
} SparseMlaParams;

/* Sparse MLA forward: examples/sparse_attention/attention.py:210-525.
 * Tensor order is the reference entry order (attention.py:211-224):
 *   q [T,H,D], ori_kv [ORI_BLOCKS,PAGE,1,D], cmp_kv [CMP_BLOCKS,PAGE/RATIO,1,D],
 *   cmp_sparse_indices i32 [T,1,TOPK], ori_block_table i32 [B,MAX_SEQ/PAGE],
 *   cmp_block_table i32 [B,MAX_SEQ/PAGE], cu_seqlens_q i32 [B+1],
 *   seqused_ori_kv i32 [B], seqused_cmp_kv i32 [B], cmp_residual_kv i32 [B],
 *   ori_topk_length i32 [T,1], sinks f32 [H], attention_out [T,H,D] (written).
 * `workspace`: NULL, or at least workspace_size_sparse_mla() bytes of device
 * memory that the call may overwrite. With a workspace and at least two work
 * items (token x BM-head tile) per compute unit, the call leaves every token's
 * selected-row list in it: at D = 512 a plan kernel writes them first and a
 * persistent attention kernel streams the items of each compute unit over
 * them, at smaller D the one-workgroup-per-item kernel writes what it resolves
 * (nothing in that call reads it: NULL is a little faster there). The plan is:
 * int32 counts [T] at byte 0 (selected rows per token), then, from byte
 * round_up(4 T, 256), uint32 lists [T][round_up(WINDOW + TOPK, 256)] of
 * tagged rows (bit 31 set: cmp_kv row, else ori_kv row; physical row in the
 * low bits) in slot order, padded with the token's first row to a multiple of
 * 32 entries (32 entries of ori_kv row 0 for an empty selection); otherwise (or with
 * params->debug_rows set) one workgroup per item (or per part of a split key,
 * params->parts, whose records a merge kernel then combines in the workspace)
 * resolves its rows itself. With one part, results are bit-identical either
 * way; split keys differ only in FP32 summation order. */
int launch_sparse_mla(void* stream, const void* q, const void* ori_kv, const void* cmp_kv,
                      const int32_t* cmp_sparse_indices, const int32_t* ori_block_table,
                      const int32_t* cmp_block_table, const int32_t* cu_seqlens_q,
                      const int32_t* seqused_ori_kv, const int32_t* seqused_cmp_kv,
                      const int32_t* cmp_residual_kv, const int32_t* ori_topk_length,
                      const float* sinks, void* attention_out, void* workspace,
                      const SparseMlaParams* params);

/* Allocation-free variant of launch_sparse_mla, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). No counterpart in the reference, whose
 * runtime owns a workspace arena per stream binding (src/runtime/kernel.py:39-49).
 * Same arguments without `workspace`: the call's workspace (row-list plan and
 * split records, workspace_size_sparse_mla bytes) lives in a static device
 * array of 32 MiB per GPU (AFA_SCRATCH_BYTES), resolved once per device; it
 * allocates nothing. Returns AFA_E_WORKSPACE, before any launch, when the
 * call's workspace exceeds it (e.g. a 32K-token prefill: 100 MiB). Results are
 * bit-identical to launch_sparse_mla with a workspace. All calls on one GPU
 * share the array: calls that overlap on one GPU (other streams, other host
 * threads) race and must be serialised by the caller. */
#define AFA_SCRATCH_BYTES (32u << 20)
int launch_sparse_mla_noalloc(void* stream, const void* q, const void* ori_kv, const void* cmp_kv,
                              const int32_t* cmp_sparse_indices, const int32_t* ori_block_table,
                              const int32_t* cmp_block_table, const int32_t* cu_seqlens_q,
                              const int32_t* seqused_ori_kv, const int32_t* seqused_cmp_kv,
                              const int32_t* cmp_residual_kv, const int32_t* ori_topk_length,
                              const float* sinks, void* attention_out, const SparseMlaParams* params);

/* Gather image of the sparse selection, the layout of the reference's gather
 * workspace and of its gather oracle (benchmarks/attention/sparse_reference.py:174-181,
 * examples/sparse_attention/gather.py:86-131, window slots from gather.py:38-60):
 *   kv_out [T,S,D] (dtype of the caches; unused slots zero),
 *   bias_out f32 [T,S] (0 selected, -inf unused).
 * Uses the fused kernel's own slot resolution and row copy. */
int launch_sparse_mla_gather(void* stream, const void* ori_kv, const void* cmp_kv,
                             const int32_t* cmp_sparse_indices, const int32_t* ori_block_table,
                             const int32_t* cmp_block_table, const int32_t* cu_seqlens_q,
                             const int32_t* seqused_ori_kv, const int32_t* seqused_cmp_kv,
                             const int32_t* cmp_residual_kv, const int32_t* ori_topk_length,
                             void* kv_out, float* bias_out, const SparseMlaParams* params);

/* Flash attention (BNSD): examples/flash_attention/attention.py:243-417.
 *   Q [B,HQ,Sq,D], K/V [B,HKV,Sk,D], O [B,HQ,Sq,D] (written).
 * The reference launcher is (stream, Q, K, V, O, workspace, Sq, Sk). */
typedef struct FaParams {
  int32_t B, HQ, HKV, D;
  int32_t dtype;   /* AFA_DTYPE_* */
  int32_t causal;  /* top-left j <= i masking (attention.py:96-110) */
  float scale;
  int32_t reserved;
} FaParams;

int launch_attention_target(void* stream, const void* Q, const void* K, const void* V, void* O,
                            void* workspace, int64_t Sq, int64_t Sk, const FaParams* params);

/* Flash attention with a workspace for calls of few query rows (decode) or
 * grids too small for the GPU: the keys are split over workgroups, whose FP32
 * partial results (per split: B * HQ * Sq rows of 128 + 2 floats) a second
 * kernel combines in split order. workspace_size_attention_target_split gives
 * the bytes a call needs (0 where one kernel does it, and then `workspace` may
 * be NULL); the launcher returns AFA_E_WORKSPACE, before any launch, for less.
 * The same results as launch_attention_target up to FP32 summation order, and
 * the same arguments accepted. launch_attention_target itself never splits. No
 * counterpart in the reference, whose operator is one kernel. */
int workspace_size_attention_target_split(uint64_t* bytes, int64_t Sq, int64_t Sk, const FaParams* params);
int launch_attention_target_split(void* stream, const void* Q, const void* K, const void* V, void* O,
                                  void* workspace, uint64_t workspace_bytes, int64_t Sq, int64_t Sk,
                                  const FaParams* params);

/* Which kernel a call of these sizes runs, with and without a workspace (the
 * launchers choose by the sizes alone): form[0] 0 for the forward kernel, 1 for
 * the kernel over packed query rows; form[1] its query rows per workgroup;
 * form[2] the key splits (1: no second kernel). For tests and profiles. */
int form_attention_target(int64_t form[3], int64_t Sq, int64_t Sk, const FaParams* params, int with_workspace);

/* Teaching attention: examples/flash_attention/simple.py:60-141.
 *   Q [H,S,128] f16, K/V [H,128,128] f16, O [H,S,128] f16 (written);
 * softmax(QK^T / sqrt(128)) normalised before the f16 cast of P. */
int launch_simple_attention(void* stream, const void* Q, const void* K, const void* V, void* O,
                            void* workspace, int64_t S, int64_t H);

/* kernel_config_<k>: cfg[5] = {tensors, runtime parameters, has_workspace,
 * compute units, SIMDs per CU} (src/backend/structured.py:619-637). */
int kernel_config_sparse_mla(int64_t cfg[5]);
int kernel_config_attention_target(int64_t cfg[5]);
int kernel_config_simple_attention(int64_t cfg[5]);

/* kernel_metadata_<k>: versioned JSON naming tensors, dtypes, shapes and
 * access modes (src/backend/abi.py:19-59). Static storage. */
const char* kernel_metadata_sparse_mla(void);
const char* kernel_metadata_attention_target(void);
const char* kernel_metadata_simple_attention(void);

/* workspace_size_<k>: bytes of the optional workspace (sparse_mla: the row-list
 * plan, T * 4 rounded up to 256 plus T * round_up(WINDOW + TOPK, 256) * 4, and
 * with K (token, BM-head tile) keys split into P parts, rounded up to 256,
 * plus K * P * (2 * BM * D + BM * BM / 2) bytes of partial results; 0 for the
 * two dense kernels); returns -1 on a NULL pointer and the
 * launcher's status for invalid sparse parameters (src/backend/workspace.py:100-130). */
int workspace_size_sparse_mla(uint64_t* bytes, const SparseMlaParams* params);
int workspace_size_attention_target(uint64_t* bytes, int64_t Sq, int64_t Sk,
                                    const FaParams* params);
int workspace_size_simple_attention(uint64_t* bytes, int64_t S, int64_t H);

/* The row-list plan alone: writes the plan that launch_sparse_mla's plan
 * kernel writes into its workspace (layout above) for every token, nothing
 * else. The counterpart of the vendor operator's metadata-preparation stage
 * (docs/operators/sparse-mla.md:10-14 in the reference); used to read the
 * selection back and to drive launch_gather_probe. `workspace` needs
 * round_up(4 T, 256) + 4 T round_up(WINDOW + TOPK, 256) bytes. */
int launch_sparse_mla_plan(void* stream, const int32_t* cmp_sparse_indices, const int32_t* ori_block_table,
                           const int32_t* cmp_block_table, const int32_t* cu_seqlens_q,
                           const int32_t* seqused_ori_kv, const int32_t* seqused_cmp_kv,
                           const int32_t* cmp_residual_kv, const int32_t* ori_topk_length, void* workspace,
                           const SparseMlaParams* params);

/* The attention over a plan alone: the persistent kernel of launch_sparse_mla
 * (one workgroup per compute unit streaming its tokens' row lists, KV ring
 * per params->ring) over the plan that launch_sparse_mla_plan wrote into
 * `workspace` for the same metadata and params. The two calls together give
 * launch_sparse_mla's output (and softmax_lse) bit for bit; the persistent
 * kernel runs here whatever T is, and no key is split. Lets a caller run the
 * plan ahead on another stream or reuse one plan for several calls over the
 * same selection. The plan must come from launch_sparse_mla_plan with the
 * same metadata and params (whether a launch_sparse_mla call wrote one depends
 * on the device and the split, so its workspace is not a plan to rely on).
 * Counts and row ids read from `workspace` are clamped to the list capacity
 * and to ori_kv / cmp_kv, so a workspace holding anything else gives a wrong
 * output but no access outside the caches. No counterpart in the
 * reference, whose operator is one kernel. Returns AFA_E_SHAPE when
 * params->debug_rows is set (the plan path writes no debug image) or no KV
 * ring fits next to the row lists (at D = 512, WINDOW + TOPK above 3328). */
int launch_sparse_mla_planned(void* stream, const void* q, const void* ori_kv, const void* cmp_kv,
                              const float* sinks, void* attention_out, const void* workspace,
                              const SparseMlaParams* params);

/* Gather probe (measurement only; the counterpart of the reference's gather
 * micro-benchmark, benchmarks/attention/gather_dma.py): streams the 1 KiB rows
 * listed in a plan (D = 512, one item per token: BM = H) from ori_kv/cmp_kv
 * through LDS as the attention kernels do, with `depth` (1, 2, 4, 6 or 8)
 * 16-row chunks in flight per workgroup and no compute, on `grid`
 * workgroups: items interleaved (balanced = 0) or an equal share of the flat
 * chunk stream each (balanced = 1, every item taken as long as item 0). Each
 * workgroup takes at most 4 items. sums [grid][16]: per thread, the sum of the
 * first dword of every row it checked (all rows streamed, mod 2^32). */
int launch_gather_probe(void* stream, const void* ori_kv, const void* cmp_kv, const void* workspace,
                        const SparseMlaParams* params, int32_t grid, int32_t depth, int32_t balanced,
                        uint32_t* sums);

/* Top-k index selection: the producer of cmp_sparse_indices, which the
 * reference takes as an input and leaves to the caller's indexer
 * (docs/operators/sparse-mla.md:8,266 in the reference). scores [T][C] f32: one
 * index score per (token, compressed position). For token t of request b
 * (cu_seqlens_q), with n queries in b, offset j and cutoff = max(0,
 * seqused_cmp_kv[b] RATIO + cmp_residual_kv[b] - n + j + 1) / RATIO (the
 * causal bound of the sparse contract, docs/operators/sparse-mla.md:41-51),
 * writes into cmp_sparse_indices [T][1][TOPK] the min(TOPK, seqused_cmp_kv[b],
 * cutoff, C) positions p < min(cutoff, C) of largest score, ascending, then
 * -1 (the input contract of docs/operators/sparse-mla.md:79). Ties go to the
 * lower position; -0 equals +0; NaN ranks above +inf. Returns AFA_E_SHAPE for
 * B, T, TOPK or C <= 0, C >= 2^31 or RATIO not 1 or 2, AFA_E_NULL for a NULL
 * pointer, before any launch. One launch; no workspace. */
typedef struct SparseTopkParams {
  int32_t B;      /* requests */
  int32_t T;      /* query tokens */
  int32_t TOPK;   /* selected positions per token (row length of the output) */
  int32_t RATIO;  /* compression ratio, 1 or 2 */
  int64_t C;      /* score columns per token (row stride of scores), < 2^31 */
} SparseTopkParams;

int launch_sparse_topk_indices(void* stream, const float* scores, const int32_t* cu_seqlens_q,
                               const int32_t* seqused_cmp_kv, const int32_t* cmp_residual_kv,
                               int32_t* cmp_sparse_indices, const SparseTopkParams* params);

/* The same selection with a workspace for few long rows (decode at long
 * contexts): each row's segments are selected by workgroups of their own, whose
 * entries a second launch merges. workspace_size_sparse_topk_indices_split gives
 * the bytes a call needs (0 where one launch does it, and then `workspace` may
 * be NULL); the launcher returns AFA_E_WORKSPACE, before any launch, for less.
 * Results are those of launch_sparse_topk_indices, value for value. */
int workspace_size_sparse_topk_indices_split(uint64_t* bytes, const SparseTopkParams* params);
int launch_sparse_topk_indices_split(void* stream, const float* scores, const int32_t* cu_seqlens_q,
                                     const int32_t* seqused_cmp_kv, const int32_t* cmp_residual_kv,
                                     int32_t* cmp_sparse_indices, void* workspace, uint64_t workspace_bytes,
                                     const SparseTopkParams* params);

/* Which form a call of these sizes runs, with and without a workspace: form[0]
 * 0 rows in registers (form[1] threads, form[2] positions per thread), 1 split
 * rows (form[1] segments per row, form[2] tokens per pair of launches), 2 the
 * filter pass, 3 the streaming passes. For tests and profiles. */
int form_sparse_topk_indices(int64_t form[3], const SparseTopkParams* params, int with_workspace);

/* Rotary positions. Pairs (u, v) of the R columns from `offset` on of every row
 * turn by the angle position * frequencies[i] (radians, float64 [R / 2]):
 *   u' = magnitude (u cos - v sin), v' = magnitude (u sin + v cos);
 * pair i is columns (i, i + R / 2) with layout 0 (halves) or (2 i, 2 i + 1) with
 * layout 1 (interleaved). inverse turns by the negative angle with the same
 * magnitude: the transposed map, which is the gradient. x and out [B][S][H][D]
 * with strides in elements, columns contiguous; the other columns are copied,
 * or, where out is x (equal strides), not touched. positions int32 or int64
 * (position_bytes 4 or 8) [S], position_stride_b elements apart for each b.
 * R up to 1024, D up to 16384. 16-byte accesses where R % 16, offset, D and the
 * strides allow them. */
typedef struct RotaryParams {
  int32_t dtype;
  int32_t layout;          /* 0 halves, 1 interleaved */
  int32_t inverse;
  int32_t position_bytes;  /* 4 or 8 */
  int32_t H, D, R, offset;
  int64_t B, S;
  int64_t x_stride_b, x_stride_s, x_stride_h;
  int64_t out_stride_b, out_stride_s, out_stride_h;
  int64_t position_stride_b;
  float magnitude;
  int32_t reserved;
} RotaryParams;

int launch_apply_rotary(void* stream, const void* x, const void* positions, const double* frequencies, void* out,
                        const RotaryParams* params);

/* Append of new tokens to a paged cache, the rotation applied on the way. Token
 * t of request b (cu_seqlens_q[b] <= t < cu_seqlens_q[b + 1]) goes to position
 * p = seqused_kv[b] - cu_seqlens_q[b + 1] + t (seqused_kv counts the new tokens,
 * as seqused_ori_kv does), row p % PAGE of page block_table[b][p / PAGE] of
 * k_cache [BLOCKS][PAGE][HKV][DK]. Its columns offset .. offset + R - 1 are
 * rotated by p as in launch_apply_rotary (R = 0: none); with `rope` [T][HKV][R]
 * they come from there, are the row's last (offset = DK - R), and k [T][HKV]
 * holds the DK - R others. v [T][HKV][DV] is copied to v_cache
 * [BLOCKS][PAGE][HKV][DV] (DV = 0: none). Strides in elements, columns
 * contiguous. Tokens at or past cu_seqlens_q[B], positions below 0 or beyond W
 * pages, and pages outside [0, BLOCKS) write nothing. No two new tokens may
 * name the same cache row. R up to 1024, DK and DV up to 16384, HKV up to 32768. */
typedef struct AppendPagedKvParams {
  int32_t dtype;
  int32_t layout;
  int32_t T, B, W, PAGE, BLOCKS;
  int32_t HKV, DK, DV, R, offset;
  int64_t k_stride_t, k_stride_h, rope_stride_t, rope_stride_h, v_stride_t, v_stride_h;
  float magnitude;
  int32_t reserved;
} AppendPagedKvParams;

int launch_append_paged_kv(void* stream, const void* k, const void* rope, const void* v, const int32_t* block_table,
                           const int32_t* cu_seqlens_q, const int32_t* seqused_kv, const double* frequencies,
                           void* k_cache, void* v_cache, const AppendPagedKvParams* params);

/* Latent attention, absorbed form, over a paged cache of rows [c | k_rope] of
 * L + R columns, kv_cache [BLOCKS][PAGE][L + R]: for token t, head h of request b
 *   s_j = scale (q[t][h] . c_j + q_rope[t][h] . k_rope_j),  out[t][h] = softmax(s) c,
 * over the rows j < seqused_kv[b], and, causal, j <= seqused_kv[b] - n + i for
 * the i-th of the request's n tokens (a length past the table's W * PAGE rows has no
 * rows there, but keeps this limit). L 128, 256 or 512, R 0 or 64, PAGE a power
 * of two from 16 on. q and out [T][H][L], q_rope [T][H][R] with strides in
 * elements (multiples of 8; rows contiguous and on 16 bytes). Rows behind
 * seqused_kv are not read; pages outside [0, BLOCKS) hold no keys; a token that
 * sees no key gets zeros; tokens at or past cu_seqlens_q[B] are left as they
 * were. softmax_lse f32 [T][H] or NULL: ln(sum_j e^(s_j)), -inf without a key.
 * Scores of a (token, head) that are NaN or overflow to +inf give NaN in both of its results.
 * Values of a row that some token of the request sees have to be finite. */
typedef struct LatentParams {
  int32_t dtype;
  int32_t causal;
  int32_t T, B, H, L, R;
  int32_t PAGE, W, BLOCKS;
  int64_t q_stride_t, q_stride_h, q_rope_stride_t, q_rope_stride_h, out_stride_t, out_stride_h;
  float scale;
  int32_t reserved;
} LatentParams;

int launch_latent_attention(void* stream, const void* q, const void* q_rope, const void* kv_cache,
                            const int32_t* block_table, const int32_t* cu_seqlens_q, const int32_t* seqused_kv,
                            void* out, float* softmax_lse, void* workspace, uint64_t workspace_bytes,
                            const LatentParams* params);

/* Bytes of device memory, on 16 bytes, that a call of these sizes needs for
 * partial results (0: none, workspace may be NULL); with less the launcher
 * returns AFA_E_WORKSPACE before any launch. Calls that may run at the same
 * time need workspaces of their own. */
int workspace_size_latent_attention(uint64_t* bytes, const LatentParams* params);

/* Which form a call of these sizes runs: form[0] packed (token, head) rows per
 * tile, form[1] workgroups that share the tiles (their keys, or, where that does not
 * pay at the lengths found on the device, whole tiles), 0 for one tile per
 * workgroup. For tests and profiles. */
int form_latent_attention(int64_t form[2], const LatentParams* params);

/* The same of a call whose tiles are shared: form[0] 1 for cache loads that stay
 * out of the caches (0: ordinary), form[1] waves that join one part of a tile, 16
 * or 1; both 0 for one tile per workgroup. Whether such a call shares keys or whole
 * tiles follows from the lengths: the 32-bit word behind its parts, at byte
 * 2 form_latent_attention[1] * form_latent_attention[0] * (L + 2) * 4 of the
 * workspace, holds the number of tiles afterwards, 0 if they stayed whole. */
int split_form_latent_attention(int64_t form[2], const LatentParams* params);

/* Latent attention, expanded form, ragged requests: for query i of the nq and
 * key j of the nk of request b, head h
 *   s_j = scale (q[i][h][0:D] . k_nope[j][h] + q[i][h][D:D+R] . k_rope[j]),  out[i][h] = softmax(s) v[:, h],
 * causal: j <= nk - nq + i. D 128, R 64. q [Tq][H][D + R], k_nope and v
 * [Tk][H][D], k_rope [Tk][R], out [Tq][H][D], strides in elements (multiples of
 * 8, rows contiguous and on 16 bytes, token strides of keys and values below
 * 2^23). softmax_lse as above, f32 [Tq][H] or NULL. */
typedef struct LatentExpandedParams {
  int32_t dtype;
  int32_t causal;
  int32_t Tq, Tk, B, H, D, R;
  int64_t q_stride_t, q_stride_h, k_stride_t, k_stride_h, k_rope_stride_t, v_stride_t, v_stride_h, out_stride_t,
      out_stride_h;
  float scale;
  int32_t reserved;
} LatentExpandedParams;

int launch_latent_attention_expanded(void* stream, const void* q, const void* k_nope, const void* k_rope, const void* v,
                                     const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, void* out,
                                     float* softmax_lse, void* workspace, uint64_t workspace_bytes,
                                     const LatentExpandedParams* params);

/* As workspace_size_latent_attention and form_latent_attention: form[0] query
 * rows per tile, form[1] key splits (1: no workspace, no second launch). */
int workspace_size_latent_attention_expanded(uint64_t* bytes, const LatentExpandedParams* params);
int form_latent_attention_expanded(int64_t form[2], const LatentExpandedParams* params);

/* Append of new tokens to a paged cache held in 8 bits, codes c of scale s
 * standing for c s. k and v [T][HKV][D] (strides in elements, columns
 * contiguous) go to the places that launch_append_paged_kv names, in k_cache and
 * v_cache [BLOCKS][PAGE][HKV][D]. GROUP tokens of a page and one head share a
 * scale, float32 k_scale and v_scale [BLOCKS][PAGE / GROUP][HKV]. With A the
 * largest finite magnitude of a block's new rows and C the largest code (448 for
 * e4m3, 127 for int8), need = 2^max(ceil(log2(A / C)), -80); a block whose first
 * row is new gets s = need, another max(need, its s), and the rows that it held
 * before the new ones are rounded anew where that is larger. Codes are x * (1 / s)
 * to nearest, ties to even, held inside [-C, C]; a NaN is e4m3's NaN, or 0. Rows
 * behind the new ones are left as they are. No two new tokens may name the same
 * row, and no two requests append to the same block. PAGE and GROUP are powers
 * of two, 16 <= GROUP <= PAGE, GROUP up to 1024, D up to 1024, HKV up to 32768,
 * T below 2^23, W * PAGE up to 2^30. */
typedef struct AppendQuantizedKvParams {
  int32_t dtype;
  int32_t code;            /* AFA_CODE_* */
  int32_t T, B, W, PAGE, GROUP, BLOCKS, HKV, D;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
} AppendQuantizedKvParams;

int launch_append_quantized_kv(void* stream, const void* k, const void* v, const int32_t* block_table,
                               const int32_t* cu_seqlens_q, const int32_t* seqused_kv, void* k_cache, void* v_cache,
                               float* k_scale, float* v_scale, const AppendQuantizedKvParams* params);

/* Attention of grouped query heads over such a cache: for token t, head h of
 * request b, with kv = h / (HQ / HKV) and the blocks' scales ks and vs
 *   s_j = scale ks_j (q[t][h] . k_j[kv]),  out[t][h] = sum_j e^(s_j) vs_j v_j[kv] / sum_j e^(s_j),
 * over the rows that launch_latent_attention names, causal or not. D 64, 128 or
 * 256, PAGE and GROUP as above. q and out [T][HQ][D] with strides in elements
 * (multiples of 8; rows contiguous and on 16 bytes). softmax_lse f32 [T][HQ] or
 * NULL. Empty rows, pages outside the cache, tokens of no request and scores
 * that are not finite as there; scales of rows that a token of the request sees
 * have to be finite and positive, and value scales below 2^-80 count as that.
 * Every key has its weight in the denominator however far the value scales lie
 * apart; values whose weight times scale is below 2^-126 of a row's largest are
 * lost from out.
 * W * PAGE up to 2^30. The workspace holds partial results; calls that may run at
 * the same time need workspaces of their own. */
typedef struct QuantizedParams {
  int32_t dtype;
  int32_t code;            /* AFA_CODE_* */
  int32_t causal;
  int32_t T, B, HQ, HKV, D;
  int32_t PAGE, GROUP, W, BLOCKS;
  int64_t q_stride_t, q_stride_h, out_stride_t, out_stride_h;
  float scale;
  int32_t reserved;
} QuantizedParams;

int launch_quantized_attention(void* stream, const void* q, const void* k_cache, const void* v_cache,
                               const float* k_scale, const float* v_scale, const int32_t* block_table,
                               const int32_t* cu_seqlens_q, const int32_t* seqused_kv, void* out, float* softmax_lse,
                               void* workspace, uint64_t workspace_bytes, const QuantizedParams* params);

/* Bytes of that workspace, on 16 bytes, and which form a call of these sizes
 * runs: form[0] packed (token, head) rows per tile (16 or 32: waves on their own,
 * 128 or 256: a workgroup of eight), form[1] key/value heads of a workgroup,
 * form[2] workgroups of the same heads that share the tiles, form[3] 1 for cache
 * loads that stay out of the caches. */
int workspace_size_quantized_attention(uint64_t* bytes, const QuantizedParams* params);
int form_quantized_attention(int64_t form[4], const QuantizedParams* params);

/* Copies page source[i] to page destination[i], i < pairs, in each of n_caches
 * tensors of BLOCKS pages (caches: device pointers, page_bytes: bytes of a page,
 * both arrays on the host). Pairs with a number outside [0, BLOCKS) copy
 * nothing. No destination may be named twice or be a source as well. Pairs times
 * the 16 KiB pieces of the largest page, up to 2^32 (what compact_pages lists is
 * far below); a call that is refused has copied nothing. */
int launch_copy_pages(void* stream, const void* const* caches, const uint64_t* page_bytes, int32_t n_caches,
                      const int32_t* source, const int32_t* destination, int32_t pairs, int32_t BLOCKS);

/* Forks requests: row b of block_table [B][W] becomes a copy of row parents[b]
 * as it was before the call, or empty (-1 throughout) where that is outside
 * [0, B). seqused_kv[b] is the length of the new row: it keeps the pages of its
 * tokens, and gets pages for `reserve` tokens more. A page that row b will go on
 * writing to (seqused_kv[b] % PAGE tokens of it are used) and that others hold
 * too is replaced by a new one, to be copied from the old: source[b],
 * destination[b], both -1 where nothing is copied. Of rows that will write to
 * one page the lowest keeps it, unless somebody else holds it. page_counts
 * [BLOCKS], the references of each page, follows all of it; free pages (count 0)
 * are handed out from the lowest up, row by row, the copy first. missing[0]
 * counts the pages that were wanted beyond the free ones or beyond the table's
 * width (2^31 - 1 at most); their entries are -1. That includes a page to be
 * copied: its row's tokens on it are lost to that row, and an entry of -1 below a
 * row's length is not wanted again by later calls. No cache is written, so that
 * block_table and page_counts saved before the call undo it. B up to 8192, BLOCKS
 * up to 2^28, PAGE a power of two. */
typedef struct ForkPagesParams {
  int32_t B, W, PAGE, BLOCKS, reserve;
} ForkPagesParams;

int workspace_size_fork_pages(uint64_t* bytes, const ForkPagesParams* params);
int launch_fork_pages(void* stream, int32_t* block_table, int32_t* page_counts, const int32_t* parents,
                      const int32_t* seqused_kv, int32_t* source, int32_t* destination, int32_t* missing,
                      void* workspace, uint64_t workspace_bytes, const ForkPagesParams* params);

/* Compacts: with n pages in use (count above 0), the k-th of those from page n on
 * is renamed to the k-th free page below n, in block_table [B][W] and in
 * page_counts [BLOCKS]; source and destination [BLOCKS / 2] list the moves, to be
 * copied, behind them -1. Afterwards pages 0 .. n - 1 are in use. */
typedef struct CompactPagesParams {
  int32_t B, W, BLOCKS;
} CompactPagesParams;

int workspace_size_compact_pages(uint64_t* bytes, const CompactPagesParams* params);
int launch_compact_pages(void* stream, int32_t* block_table, int32_t* page_counts, int32_t* source, int32_t* destination,
                         void* workspace, uint64_t workspace_bytes, const CompactPagesParams* params);

/* Measurement helpers (no reference kernel; the reference sweeps a >= 4x L2
 * buffer before each timed launch, benchmarks/cache.py:13-92 and
 * benchmarks/cache_sweep.py:15-32). Reads `bytes` of `buffer` through the
 * caches (cached 16-byte loads, nothing written back for a zero-filled
 * buffer) so that the next launch starts cold. */
int launch_cache_flush(void* stream, void* buffer, uint64_t bytes);

/* Measurement helper (no reference kernel): runs `spins` dependent FMAs in
 * every thread of 1024 workgroups of 256 (every SIMD busy) and writes, from
 * workgroup 0, out[0..1] = the shader-cycle counter before and after and
 * out[2..3] = the 100 MHz real-time counter before and after (out has 5
 * entries): the shader clock is 100 MHz x (out[1] - out[0]) / (out[3] - out[2]). */
int launch_clock_probe(void* stream, uint64_t* out, int32_t spins);

/* Library version string. */
const char* ascendflow_amd_version(void);

#ifdef __cplusplus
}
#endif

#endif /* ASCENDFLOW_AMD_H */
