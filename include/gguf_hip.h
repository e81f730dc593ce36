/* gguf_hip.h - C ABI of the MI355X (gfx950) GGUF quantized linear path.
 *
 * A drop-in for the out-of-tree vLLM GGUF plugin's linear path: the entry points below are
 * what that plugin's Python binds for (a) dequantize(W, type, shape), (b) the load-time tile
 * repack and grouped-layer preparation, and (c) the grouped matmul op called from
 * GGUFLinearMethod.apply(layer, x, bias).  Plain C: raw device pointers, sizes and a HIP stream
 * passed as void*.  No allocation happens inside any entry point: outputs, tiles and workspace
 * are owned by the caller (torch), and every launch goes on the caller's stream.
 *
 * Status: every int-returning function returns GQK_OK (0) or a negative GQK_ERR_* code;
 * gqk_last_error() returns a thread-local message for the last failure on the calling thread.
 */
#ifndef GGUF_HIP_H
#define GGUF_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GQK_OK 0
#define GQK_ERR_TYPE (-1)  /* GGML type without a kernel (reference: NotImplementedError,
                              gguf-plugin/gluon/interface.py:78-79) */
#define GQK_ERR_SHAPE (-2) /* shape / size / alignment contract broken (reference: AssertionError,
                              gguf-plugin/gluon/tiles_grouped.py:1211-1263) */
#define GQK_ERR_FORM (-3)  /* plan does not serve this launch (M outside the plan's range) */
#define GQK_ERR_HIP (-4)   /* HIP runtime error at launch */
#define GQK_ERR_ARG (-5)   /* null pointer or bad argument */

#define GQK_FORM_GEMV 1 /* M <= 32, every type: streaming forms over (tile, k-range) rows: the in-register
                           decode GEMV up to 16 rows (small shards up to 8 rows in its slab form,
                           plan bm = 2: a row per 32-row slab over the whole k-range), the mid form
                           (g = 8) for 17..32 (small shards at 9..32 rows in its slab form, bm = 2) */
#define GQK_FORM_GEMM 2 /* M > 32: dequant bf16 MFMA GEMM, weights decoded in registers (any M) */

#define GQK_CTR_BYTES 262144 /* the arrival-counter region at the start of every workspace */

#define GQK_DTYPE_F32 0
#define GQK_DTYPE_BF16 1
#define GQK_DTYPE_F16 2
#define GQK_DTYPE_FP8 3 /* OCP e4m3 (pages of a key-value cache) */

/* One shard of a grouped layer: its rows sit at byte `offset` of the packed tile buffer. */
typedef struct gqk_shard {
  int32_t ggml_type;
  int32_t reserved;
  int64_t n;      /* output rows */
  int64_t offset; /* byte offset of the shard's tiles in the packed buffer */
} gqk_shard;

/* Launch plan of a grouped layer for one batch-row bucket (filled by gqk_plan). */
typedef struct gqk_plan_info {
  int32_t form;       /* GQK_FORM_GEMV or GQK_FORM_GEMM */
  int32_t m_max;      /* largest batch rows M the plan serves (GEMV: 4 * g) */
  int32_t g;          /* GEMV: groups of 4 tokens (1, 2, 4; 8 = the mid form, 17..32 rows, or its slab
                         form from 9 rows) */
  int32_t bm;         /* GEMM: the row-count class (64, 128, 256: two, two, four 64-row tiles per
                         descriptor row; the launch picks its tile geometry from it); GEMV (g <= 2): 1 when every wave streams
                         exactly one 256-weight record (the launch takes the pipeline-free kernel),
                         2 for the slab form (a workgroup per 32-row half tile over the whole k-range,
                         one wave per pair of super-blocks, no split-K partials; with g = 8 the mid
                         form's slab) */
  int32_t split;      /* GEMV: most workgroups sharing one tile (partials summed in split order in-kernel when > 1) */
  int32_t n_desc;     /* descriptor rows (workgroups along N x K) */
  int32_t types_mask; /* the GGML type of every shard, or 0 when the shards mix types */
  int32_t nb;         /* K / 256 */
  int32_t nw;         /* GEMV: waves per workgroup (they split the workgroup's k-range) */
  int32_t ctr_bytes;  /* bytes of arrival counters at the start of the workspace: GQK_CTR_BYTES in
                         every plan, so one workspace serves every layer and every M */
  int64_t n_total;    /* output columns: sum of the shards' rows */
  int64_t workspace_bytes; /* device workspace gqk_linear needs (any M <= m_max) */
} gqk_plan_info;

/* Last error message of the calling thread ("" when none). */
const char* gqk_last_error(void);

/* Library version: major * 10000 + minor * 100 + patch. */
int gqk_version(void);

/* Host-only metadata of a GGML type: info[0..3] = weights per block, bytes per block, bytes per
 * 256 weights, number of tile planes; planes (if not NULL, 6 ints per plane) = bytes per row,
 * segments, first raw offset, segment bytes, segment stride, column width of the tile layout.  Replaces the reference's tile
 * registry TILE_TYPES (gguf-plugin/gluon/tiles.py:24-36) and gguf.GGML_QUANT_SIZES. */
int gqk_type_info(int ggml_type, int32_t* info, int32_t* planes);

/* Dequantize n rows of K weights of `ggml_type` (raw GGUF blocks, row stride in bytes) into
 * out[n, ld_out] of out_dtype (GQK_DTYPE_*): fp32 bit-exact with gguf-py's dequantizer, bf16 /
 * fp16 the round-to-nearest-even of it.  Replaces ops.ggml_dequantize(W, type, m, n, dtype)
 * (gguf-plugin/patches/gguf-prefill-dispatch.patch:42-45, gguf-plugin/gluon/tiles.py:147-149). */
int gqk_dequantize(const void* W, int64_t w_row_stride, int ggml_type, int64_t n, int64_t K, void* out,
                   int64_t ld_out, int out_dtype, void* stream);

/* Dequantize n rows of K weights straight from the tile layout (gqk_repack's output) into
 * out[n, ld_out] of out_dtype, in one pass (no raw-row temporary); the same bits as
 * gqk_dequantize of the raw rows.  Replaces dequantize_tiles / dequantize_iq3s_tiles
 * (gguf-plugin/gluon/tiles.py:141-149, gguf-plugin/gluon/iq3s_tile_dequant.py:22-63). */
int gqk_dequantize_tiles(const void* tiles, int ggml_type, int64_t n, int64_t K, void* out, int64_t ld_out,
                         int out_dtype, void* stream);

/* Bytes of the tile layout of an n x K shard (< 0: error code).  K % 256 == 0. */
int64_t gqk_tiles_bytes(int ggml_type, int64_t n, int64_t K);

/* Raw GGUF rows -> CDNA4 plane-major tiles (64-row tiles x 256-weight super-blocks, rows past n
 * zero).  Replaces repack_tiles (gguf-plugin/gluon/tiles.py:128-130). */
int gqk_repack(const void* W, int64_t w_row_stride, int ggml_type, int64_t n, int64_t K, void* tiles, void* stream);

/* Tiles -> raw GGUF rows (bit-exact inverse of gqk_repack).  Replaces unrepack_tiles
 * (gguf-plugin/gluon/tiles.py:56-67). */
int gqk_unrepack(const void* tiles, int ggml_type, int64_t n, int64_t K, void* W, int64_t w_row_stride, void* stream);

/* Host code (no launch, no allocation): the launch plan of a grouped layer (shards packed back to
 * back, all of K columns) for batch rows M: fills *info and, if desc is not NULL and
 * desc_capacity (int32 words) is enough, the descriptor table (16 int32 per row) to upload to
 * the device.  cus: compute units of the device the plan is for (256 on MI355X); 0 asks the HIP
 * runtime for the current device's count (initialising the runtime; 256 when no device is
 * visible).  target_wgs > 0 overrides the GEMV heuristic's target of resident waves (0 = eight per
 * CU), from which the waves per workgroup and the split-K factor follow.  GEMM plans (M > 32)
 * take their descriptor rows from M and, at 129..384 rows (129..768 for K <= 8192), from the layer's
 * size against the CU count.  Replaces prepare_grouped_layer / descriptors / grouped_split_for
 * (gguf-plugin/gluon/tiles_grouped.py:237-299). */
int gqk_plan(const gqk_shard* shards, int nshards, int64_t K, int M, int target_wgs, int cus, int32_t* desc,
             int64_t desc_capacity, gqk_plan_info* info);

/* Device workspace bytes gqk_linear needs for this plan at M batch rows (0: none; < 0: error).
 * GEMV plans with split-K need info->workspace_bytes; GEMM plans need room for their stream-K
 * partial tiles, which depends on M and on the current device's CU count.  Replaces the reference's transient split-K partials (gguf-plugin/gluon/tiles_grouped.py:1233-1238). */
int64_t gqk_linear_workspace_bytes(const gqk_plan_info* info, int M);

/* The tile geometry and schedule gqk_linear takes for a GEMM plan at M batch rows on a device of `cus`
 * compute units (0: the current device), on the host: out[7] = 32-token blocks per tile, 32-row blocks
 * per tile, k-groups of waves, k-splits per tile (workgroups; 1 for the persistent form of 8 x 8 blocks),
 * workgroups of the persistent form's remainder tiles, workgroups launched, fp32 partial slots.  For
 * tests and measurements; no counterpart in the reference. */
int gqk_gemm_pick(const gqk_plan_info* info, int M, int cus, int32_t* out);

/* Workspace bytes that serve every GEMM plan at any M on the current device (< 0: error): one
 * buffer of this size (or of a layer's GEMV workspace_bytes, if larger) serves every layer on the
 * device, as calls on one stream never overlap.  No counterpart in the reference, whose split-K
 * partials are transient torch tensors (gguf-plugin/gluon/tiles_grouped.py:1233-1238). */
int64_t gqk_workspace_bytes_max(void);

/* Measurement only, no counterpart in the reference: a plain streaming read of `bytes` (a
 * multiple of 1 KiB, at most 2 GiB) at `buf` on `grid` workgroups of `waves` (1..16) waves, each
 * wave reading one contiguous share and writing one folded word to sink[wave] (grid * waves
 * uint32 words).  Timed over a shard's packed bytes on the shard's own grid it gives the memory
 * floor that bench.py reports beside each launch. */
int gqk_read_floor(const void* buf, int64_t bytes, int grid, int waves, void* sink, void* stream);

/* y[M, ldy] (bf16) = x[M, ldx] (bf16) @ W^T (+ bias) over the grouped layer's shards (columns in
 * shard order), on `stream`.  bias: NULL or bf16 [info->n_total] device memory, added in fp32
 * before the single rounding to bf16 (the reference adds it afterwards with out.add_(bias),
 * gguf-plugin/patches/gguf-tiles-grouped.patch:167-168).  desc_dev: the plan's descriptor table in device memory.  workspace: at
 * least gqk_linear_workspace_bytes(info, M) bytes of 256-byte aligned device memory (NULL when
 * that is 0) holding arrival counters (its first GQK_CTR_BYTES bytes) and fp32 partials (after
 * them); it must be zero-filled before its first use, every launch leaves the counters at zero
 * again, one workspace serves every plan of every layer (the counter region is the same in all
 * of them), and launches sharing one workspace must not overlap in time.  M must be <= info->m_max.  Replaces the grouped op
 * torch.ops.vllm._fused_mul_mat_gguf_tiles_grouped -> gluon_mul_mat_tiles_grouped
 * (gguf-plugin/patches/gguf-tiles-grouped.patch:28-72, gguf-plugin/gluon/interface.py:141-188). */
int gqk_linear(const void* packed, const int32_t* desc_dev, const gqk_plan_info* info, const void* x, int64_t ldx,
               int M, void* y, int64_t ldy, const void* bias, void* workspace, int64_t workspace_bytes, void* stream);

/* gqk_linear without a workspace argument, for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).  No counterpart
 * in the reference.  The split-K / stream-K counters and partials live in a file-scope device
 * array of GQK_NOALLOC_SCRATCH_BYTES per GPU (held until the process ends; its address is taken
 * once per device on the first call, which also clears its counters with a fill kernel on
 * `stream`).  Allocates nothing.  A plan that needs more workspace at this M is refused with
 * GQK_ERR_SHAPE: GEMM launches above 128 rows with many remainder tiles, and GEMV plans whose split-K partials
 * exceed the 32 MiB (those are 64 rows x m_max tokens x 4 bytes per partial slot: at most 4,096
 * slots at m_max = 32, 8,192 at 16, 32,768 at 4; e.g. a layer of 2,374 tiles at K = 16384 split 16
 * ways at M <= 4 needs ~39 MB).  Every call on one GPU shares that
 * GPU's array: calls that overlap in time on one GPU (other streams, other threads) race. */
#define GQK_NOALLOC_SCRATCH_BYTES (GQK_CTR_BYTES + 33554432)
int gqk_linear_noalloc(const void* packed, const int32_t* desc_dev, const gqk_plan_info* info, const void* x,
                       int64_t ldx, int M, void* y, int64_t ldy, const void* bias, void* stream);

/* ---- around the linear path: what a decode step does with its outputs ----------------------------
 * No counterpart in the reference's plugin, which leaves these to the server it is loaded into.
 * Contents of device arrays are checked where they are read: an index out of its range reads nothing
 * and makes the token's result NaN (a slot out of range stores nothing). */

/* Low-rank adapters of many requests beside a shared projection, M rows (at most GQK_LORA_MAX_ROWS):
 *   out[m, n] = y[m, n] + scales[i] * sum_r b[i, n, r] * sum_k a[i, p(n), r, k] * x[m, k],  i = ids[m]
 * p(n): the part (q, k, v; gate, up) of column n, parts side by side with n_outs[p] columns each.  A row with a
 * negative id gets y; one with an id >= slots NaN.  y, x, out: bf16 or fp16 (dtype) rows of any stride,
 * out may be y or x; a [slots, parts, rank, K] and b [slots, sum(n_outs), rank] of the same type, contiguous, K and
 * rank multiples of 8, rank <= 256 (adapters of a lower rank are padded with zeros), parts <= 8; ids
 * int32 [M], or int64 with ids_64; scales fp32 [slots] or NULL (1).  x, a, b are 16-byte aligned.  Products
 * and sums are in fp32, rounded once to out.  K and x's row stride (where M > 1) are at most GQK_LORA_MAX_K.
 * workspace: gqk_lora_workspace_bytes bytes, 256-byte aligned (fewer rows may want more: K is cut finer); in a smaller one, down to
 * GQK_CTR_BYTES + 4 M parts rank, K is cut into fewer splits.  Its first GQK_CTR_BYTES are left alone, so that a linear layer's
 * workspace serves (calls in stream order). */
#define GQK_LORA_MAX_K 4194296 /* 256 rows stay below 2^31 bytes */
#define GQK_LORA_MAX_ROWS 4194240 /* 65535 blocks of 64 */
int64_t gqk_lora_workspace_bytes(int M, int64_t K, int parts, int rank);
int gqk_lora_add(const void* y, int64_t y_row, const void* x, int64_t x_row, int M, int64_t K, const void* a,
                 const void* b, int slots, int parts, const int64_t* n_outs, int rank, const void* ids, int ids_64,
                 const float* scales, int dtype, void* out, int64_t out_row, void* workspace, int64_t workspace_bytes,
                 void* stream);

/* The pages of one layer's key-value cache: k and v as [pages, page_size, heads, dim] with any strides
 * (in elements, multiples of 8, at most GQK_MAX_PAGE_STRIDE and of tokens GQK_MAX_TOKEN_STRIDE; dims side by side), so that a token's heads or a head's tokens may lie together.
 * dtype: the heads' own type, or GQK_DTYPE_FP8, whose values stand for themselves times k_scale / v_scale
 * (fp32 [heads] in device memory, NULL: 1).  Pages are aligned to 8 elements. */
#define GQK_MAX_PAGE_STRIDE 2147483640
#define GQK_MAX_TOKEN_STRIDE 33554432
typedef struct gqk_pages {
  void* k;
  void* v;
  int64_t k_page, k_token, k_head;
  int64_t v_page, v_token, v_head;
  const float* k_scale;
  const float* v_scale;
  int32_t dtype, pages, page_size, heads, dim;
} gqk_pages;

/* Heads of one token after the other: [tokens, heads, dim] with strides in elements (multiples of 8; data 16-byte
 * aligned, dims side by side): e.g. a column range of qkv's output. */
typedef struct gqk_heads {
  void* data;
  int64_t row, head;
  int32_t heads;
} gqk_heads;

#define GQK_ROPE_UNIT_OFFSET 1 /* norm weights are 1 + w */
#define GQK_ROPE_INTERLEAVED 2 /* rotated pairs are dims (2 i, 2 i + 1), not (i, i + rot / 2) */

/* RMS norm of each head of q and k (weights [dim] of the heads' type or fp32; NULL: no norm), then the rotation of
 * its first rot dims by the token's position: table fp32 [table_rows, rot] = cos | sin of each pair's angle.  One
 * launch; arithmetic in fp32, rounded once.  out_q / out_k may be q / k themselves (or NULL for out_k when the
 * keys are only stored; k NULL: queries alone).  With pages, token t's keys and values (v, not changed) are stored at slot
 * slots[t] = page * page_size + place (negative: not stored); in fp8 pages as value / scale, at most 448 in size.
 * dim: a multiple of 8 up to 256, rot even; positions and slots int32, or int64 where the _64 flag is set.  A position
 * outside of the table makes the token's heads NaN. */
int gqk_qk_norm_rope(const gqk_heads* q, const gqk_heads* k, const gqk_heads* v, int dtype, int64_t tokens, int dim,
                     const void* positions, int positions_64, const float* table, int64_t table_rows, int rot,
                     const void* q_weight, const void* k_weight, int weight_dtype, float eps, int flags,
                     const gqk_heads* out_q, const gqk_heads* out_k, const gqk_pages* pages, const void* slots,
                     int slots_64, void* stream);

/* Attention of one new token per sequence over its pages, split over the length (one launch; a second one joins more than
 * 16 splits of a sequence, or those of many heads that share one of keys):
 *   out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j,   key j of sequence b in page table[b, j / page_size]
 * over j in [max(0, lengths[b] - window), lengths[b]) (window 0: all).  No key (a length of zero or less): zeros, lse -inf;
 * a length above max_length, or a page outside of the cache among the keys: NaN.  Query head h reads key head h / (q_heads / heads).  q, out: bf16 or fp16
 * [batch, q_heads, dim]; table int32 [batch, table_width] with rows table_row apart; lse: NULL or fp32
 * [batch, q_heads], log sum_j exp.  Scores, softmax and sums are in fp32; the probabilities that multiply v are rounded to
 * the heads' type.  workspace: gqk_paged_attention_workspace_bytes bytes, 256-byte aligned, zeroed
 * before its first use (arrival counters, which every launch leaves at zero, and fp32 partials); in a smaller one (or none: NULL)
 * the length is cut into fewer splits.  A linear layer's workspace serves (calls in stream order). */
#define GQK_MAX_KEYS 0x7ffffc00 /* the largest max_length */
int64_t gqk_paged_attention_workspace_bytes(int batch, int q_heads, int kv_heads, int dim, int max_length, int window);
int gqk_paged_attention(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads,
                        const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width,
                        const int32_t* lengths, int max_length, int window, float scale, void* out, int64_t out_row,
                        int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream);

/* gqk_paged_attention with a table for each key head: key j of sequence b, for the query heads of key head h, lies in page
 * table[b, h, j / page_size], the rows of one sequence's heads table_head apart (0: one for all).  lengths[b] counts the keys that each head's row lists. */
int gqk_paged_attention_heads(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads,
                              const gqk_pages* pages, const int32_t* table, int64_t table_row, int64_t table_head, int table_width,
                              const int32_t* lengths, int max_length, int window, float scale, void* out, int64_t out_row,
                              int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- steps of several new tokens per sequence ------------------------------------------------- */

/* What a step needs to know of its tokens, from the sequences' lengths.  Sequence b of the batch is request requests[b] (int32, or int64
 * with requests_64; negative: no sequence), whose pages are lists[requests[b], :] (int32 [lists_n, width], rows list_row apart); it has
 * lengths[b] keys in the cache and brings counts[b] new tokens, which are rows starts[b] .. starts[b + 1] of the step's `tokens` rows
 * (one sequence's after another's).  Written:
 *   table [batch, width]      the pages of lengths[b] + counts[b] keys, -1 behind them
 *   totals [batch]            lengths[b] + counts[b]
 *   starts [batch + 1]
 *   sequences [tokens]        the row's sequence, -1 behind the last
 *   positions [tokens]        lengths[b] + i for new token i; in a tree lengths[b] + the number of its ancestors (0 behind the last)
 *   slots [tokens] (int64)    page * page_size + place of key lengths[b] + i (-1 behind the last, and where the list has a negative page)
 *   mask [tokens, (tree + 31) / 32]   with parents: the bits of the token's ancestors and its own
 * parents: NULL (a chain), or int32 [tokens], the number of each new token's parent among its sequence's (-1: the cache's last key), which comes before
 * it; tree: the most new tokens of a sequence then (at most GQK_MAX_TREE), else 0.  What cannot be (a request that has no list, lengths beyond
 * its width or negative, more tokens than rows or than `tree`): totals 2^31 - 1, for which the attention answers NaN, no slots, positions -1;
 * a parent that does not come before its child: an empty mask and position -1 for the token and those below it. */
#define GQK_MAX_TREE 1024
int gqk_step_tables(const int32_t* lists, int64_t list_row, int lists_n, int width, const void* requests, int requests_64,
                    const int32_t* lengths, const int32_t* counts, int batch, int tokens, int page_size, const int32_t* parents, int tree,
                    int32_t* table, int32_t* totals, int32_t* starts, int32_t* sequences, int32_t* positions, int64_t* slots, int32_t* mask,
                    void* stream);

/* The residual's addition and the RMS norm of rows x [rows, dim] (bf16 or fp16, rows x_row elements apart, any dim up to
 * GQK_NORM_MAX_DIM):
 *   s = x + residual,  out_residual = s,  out = s rsqrt(mean(s^2) + eps) * weight
 * residual NULL: s = x; out_residual NULL: not written; weight NULL: 1, else [dim] of x's type or fp32, 1 + weight with
 * GQK_ROPE_UNIT_OFFSET.  Arithmetic is in fp32, the norm that of s before it is rounded.  out_dtype: x's, or
 * GQK_DTYPE_FP8: out = the values divided by scale, which is fp32 [rows], or [rows, dim / group] with a group (a power of two from 32
 * to 512 that divides dim): the largest size of a value (2^-100 at least) / 448.  out, out_residual may be x, residual (whole, with their row strides);
 * out in 8 bits shares no memory with the inputs,
 * and the outputs none with each other. */
#define GQK_NORM_MAX_DIM 32768
int gqk_add_rms_norm(const void* x, int64_t x_row, const void* residual, int64_t residual_row, int dtype, int64_t rows, int dim,
                     const void* weight, int weight_dtype, float eps, int flags, void* out, int64_t out_row, int out_dtype, float* scale,
                     int group, void* out_residual, int64_t out_residual_row, void* stream);

/* Attention of several new tokens per sequence over its pages.  q, out: [tokens, q_heads, dim], sequence b's tokens the rows starts[b] ..
 * starts[b + 1] (int32 [batch + 1]; rows outside of them, and a sequence whose rows are not within q's, are not written); lengths[b] counts its
 * keys, the new tokens' among them, which are its last ones in their order.  New token i sees the keys before the new
 * ones, and of those the ones that its mask names: bit j % 32 of mask[starts[b] + i, j / 32] (int32 [tokens, mask_words]) is new token j; mask
 * NULL: new tokens 0 .. i.  window > 0: of the keys that it sees the last `window`.  No key: zeros, lse -inf.  A length above max_length or below the
 * sequence's new tokens, more of them than max_tokens or the mask's bits: NaN for the sequence; a page outside of the cache: NaN for the tokens whose
 * keys it would hold, and maybe for others of the sequence; entries of pages that lie behind the windows of all the sequence's tokens are not looked
 * at.  Values that are not finite at keys that a token does not see do not reach it.  Everything else as gqk_paged_attention (one launch, a second where
 * the keys are split).  Refused: tokens q_heads / 64 + batch heads of 2^24 or more (128 for 64 where a sequence may have more than 64 rows
 * of a key head), which are more than a launch takes. */
#define GQK_MAX_TOKENS 1048576
#define GQK_MAX_GROUP 1024 /* query heads of a key head */
int64_t gqk_tree_attention_workspace_bytes(int tokens, int batch, int q_heads, int kv_heads, int dim, int max_tokens, int max_length,
                                           int window);
int gqk_tree_attention(const void* q, int64_t q_row, int64_t q_head, int dtype, int tokens, int batch, int q_heads,
                       const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths,
                       const int32_t* starts, const int32_t* mask, int mask_words, int max_length, int max_tokens, int window, float scale,
                       void* out, int64_t out_row, int64_t out_head, float* lse, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- the pages of a long cache that are worth reading ------------------------------------------ */

/* Bounds of the keys in the pages that hold each sequence's last `count` keys, [pages, 2, heads, dim] of the pages' type (contiguous, aligned to 8 elements): the
 * smallest and the largest of the page's keys of this sequence, per head and dim (NaN for both where one is NaN).  Only pages->k and its strides are read.  Pages
 * that several sequences hold must hold the same keys of each; a length or page out of its range writes nothing. */
int gqk_page_bounds(const gqk_pages* pages, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths, int batch,
                    int count, void* bounds, void* stream);

/* For each sequence and key head the `keep` pages of its table to attend to: the first `sink`, the last `recent` (one at least), and of the others
 * those with the largest  max over the key head's query heads of sum_d max(q_d lo_d, q_d hi_d), which no key of the page exceeds; among equals the first.
 * out [batch, heads, keep]: their pages in the table's order (-1 behind them, where a sequence has fewer), out_lengths [batch]: the keys in them (the last
 * page alone may be partial), for gqk_paged_attention_heads.  The order is that of the scores in 64 bits; a score that is NaN counts as infinity.
 * Positive scales of 8-bit keys do not change it.  A page outside of the cache is taken (the attention then answers NaN), a length above max_length
 * gives 2^31 - 1.  workspace: gqk_select_pages_workspace_bytes bytes, 256-byte aligned, or less, down to one sequence's (they then go in
 * turns); its first GQK_CTR_BYTES are left alone. */
int64_t gqk_select_pages_workspace_bytes(int batch, int heads, int page_size, int max_length);
int gqk_select_pages(const void* q, int64_t q_row, int64_t q_head, int dtype, int batch, int q_heads, const void* bounds, int bounds_dtype,
                     int pages, int heads, int dim, const int32_t* table, int64_t table_row, int table_width, const int32_t* lengths,
                     int max_length, int page_size, int keep, int sink, int recent, int32_t* out, int32_t* out_lengths, void* workspace,
                     int64_t workspace_bytes, void* stream);

/* Page src[i] to page dst[i] in each of `planes` planes (a layer's keys, a layer's values, ...), for n pairs: page p of
 * plane l is the page_bytes bytes at base + l * plane_stride + p * page_stride.  src and dst are host arrays, read
 * before the call returns (a captured graph copies the pairs of its capture).  A page outside of
 * the cache, one that is written twice, or one that is both read and written is refused (GQK_ERR_SHAPE, GQK_ERR_ARG) and
 * nothing is copied. */
int gqk_copy_pages(void* base, int64_t planes, int64_t plane_stride, int64_t pages, int64_t page_stride,
                   int64_t page_bytes, const int32_t* src, const int32_t* dst, int64_t n, void* stream);

/* ---- GGUF v3 files: the load path ----------------------------------------------------------
 * The reference's tensors come from vLLM's GGUF loader (gguf-py 0.17.1 GGUFReader,
 * gguf-plugin/requirements.txt:1) and are repacked at load time by _create_tiles
 * (gguf-plugin/patches/gguf-tiles-all-types.patch:59-131).  Here a C++ reader maps the file read
 * only; tensor data is never copied on the host. */
typedef struct gqk_gguf gqk_gguf; /* an open GGUF file (immutable: safe to share across threads) */

/* GGUF metadata value types */
#define GQK_GGUF_UINT8 0
#define GQK_GGUF_INT8 1
#define GQK_GGUF_UINT16 2
#define GQK_GGUF_INT16 3
#define GQK_GGUF_UINT32 4
#define GQK_GGUF_INT32 5
#define GQK_GGUF_FLOAT32 6
#define GQK_GGUF_BOOL 7
#define GQK_GGUF_STRING 8
#define GQK_GGUF_ARRAY 9
#define GQK_GGUF_UINT64 10
#define GQK_GGUF_INT64 11
#define GQK_GGUF_FLOAT64 12

typedef struct gqk_gguf_tensor {
  const char* name;   /* NUL-terminated, owned by the handle */
  int32_t ggml_type;
  int32_t n_dims;
  int64_t dims[4];    /* GGUF order: dims[0] = weights per row (K), dims[1] = rows (N); unused = 1 */
  int64_t offset;     /* absolute byte offset of the data in the file */
  int64_t nbytes;     /* packed bytes; -1 for a type without a fixed block size here */
  const void* data;   /* host pointer into the read-only mapping (NULL when nbytes < 0) */
} gqk_gguf_tensor;

typedef struct gqk_gguf_kv {
  const char* key;    /* NUL-terminated, owned by the handle */
  int32_t type;       /* GQK_GGUF_* */
  int32_t array_type; /* element type of an ARRAY */
  int64_t count;      /* 1 for a scalar, bytes of a STRING, elements of an ARRAY */
  int64_t i64;        /* integer and BOOL scalars (UINT64 as its bit pattern) */
  double f64;         /* FLOAT32 / FLOAT64 scalars */
  const void* data;   /* STRING bytes (not NUL-terminated) or the first ARRAY element (mapping) */
} gqk_gguf_kv;

/* (weights per block, bytes per block) of a GGML type: gguf.GGML_QUANT_SIZES
 * (gguf-plugin/patches/gguf-prefill-dispatch.patch:42-45 reads it for the dequant shape). */
int gqk_ggml_type_size(int ggml_type, int32_t* block, int32_t* bytes);

/* Map and parse a GGUF v3 file (GGUFReader(path) in gguf-py).  *out is NULL on failure. */
int gqk_gguf_open(const char* path, gqk_gguf** out);
void gqk_gguf_close(gqk_gguf* f);
/* Counts, alignment (general.alignment, default 32), data-section offset and version. */
int gqk_gguf_info(const gqk_gguf* f, int64_t* n_tensors, int64_t* n_kv, int64_t* alignment, int64_t* data_offset,
                  int32_t* version);
/* Tensor info i (GGUFReader.tensors[i]); index of a tensor by name, -1 when absent. */
int gqk_gguf_tensor_at(const gqk_gguf* f, int64_t i, gqk_gguf_tensor* out);
int64_t gqk_gguf_find_tensor(const gqk_gguf* f, const char* name);
/* Metadata key/value i (GGUFReader.fields); index of a key, -1 when absent; string j of a STRING
 * (j = 0) or of an ARRAY of strings. */
int gqk_gguf_kv_at(const gqk_gguf* f, int64_t i, gqk_gguf_kv* out);
int64_t gqk_gguf_find_kv(const gqk_gguf* f, const char* key);
int gqk_gguf_kv_string(const gqk_gguf* f, int64_t i, int64_t j, const char** s, int64_t* len);

/* Load path of one quantized matrix: its raw rows from the mapping into `staging` (device, at
 * least nbytes), then gqk_repack into `tiles` (gqk_tiles_bytes(type, dims[1], dims[0]) bytes), both
 * on `stream`.  The copy reads pageable host memory, so it returns once the rows are staged. */
int gqk_gguf_upload_tiles(const gqk_gguf* f, int64_t i, void* staging, int64_t staging_bytes, void* tiles,
                          void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GGUF_HIP_H */
