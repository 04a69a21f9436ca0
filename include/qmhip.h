/* qmhip.h -- C-ABI of the MI355X (gfx950) HIP token loop for quillm.
 *
 * Plain C: pointers, sizes and int return codes; no C++ or torch types. Every entry point
 * names the reference interface it stands in for (file:line in the reference tree).
 *
 * Conventions (mirroring the reference's, see its src/model.h:32-36 and src/ops.h:23-34):
 *   - op-level functions take DEVICE pointers and a stream (NULL = the library's stream) and
 *     return 0, or -1 with a message in qmh_last_error(). They are asynchronous on the stream.
 *   - model-level functions take host arguments; forward returns model-owned (pinned host)
 *     logits, valid until the next call, or NULL on a bad token/pos, like the reference.
 *   - results are bitwise identical to the reference's scalar ISA path
 *     (src/kernels_scalar.c) and bitwise reproducible run to run.
 *   - nothing here allocates on the host heap per token; device memory is allocated at
 *     model creation only.
 */
#ifndef QMHIP_H
#define QMHIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* tensor dtypes, same codes as the reference's qm_dtype (src/qm_base.h:11-15) */
enum { QMH_F32 = 0, QMH_Q8_0 = 2, QMH_Q4_0 = 3 };
/* 16-bit element types of rows, pages and logits, for the ops of "several continuations of one prompt"
 * below only: no weight and no file has them. No reference counterpart. */
enum { QMH_F16 = 1, QMH_BF16 = 4 };

/* ------------------------------------------------------------------ runtime */

/* 1 if a gfx950 device is visible. Stands in for qm_cpu_supports(QM_ISA_HIP) next to the
 * ISA probe of src/cpu.c:39-49. */
int qmh_available(void);
/* Select a device and create the library stream. 0 or -1. Stands in for qm_kernels_select
 * (src/kernels_scalar.c:71-76) for the "hip" ISA. */
int qmh_init(int device);
/* Thread-local message for the last -1/NULL return. */
const char *qmh_last_error(void);
/* The library's HIP stream (a hipStream_t) -- lets callers order their own work after ours. */
void *qmh_stream(void);

/* device memory plumbing for callers that hold no HIP runtime of their own */
void *qmh_dev_alloc(size_t bytes);
int qmh_dev_free(void *p);
int qmh_memcpy_h2d(void *dst, const void *src, size_t bytes);
int qmh_memcpy_d2h(void *dst, const void *src, size_t bytes);
int qmh_memset(void *dst, int value, size_t bytes);
int qmh_sync(void);

/* ------------------------------------------------------------------ op level (device pointers) */

/* fp16 <-> fp32, elementwise over n values. qm_fp16_to_fp32 / qm_fp32_to_fp16 (src/fp16.c:6-56) */
int qmh_fp16_to_fp32(const uint16_t *h, float *f, int64_t n, void *stream);
int qmh_fp32_to_fp16(const float *f, uint16_t *h, int64_t n, void *stream);

/* rows x n floats -> rows rows of Q8_0 / Q4_0 blocks in the reference byte layout (34 / 18 B
 * per 32 values, zero padded). qm_quantize_row_q8 / qm_quantize_row_q4 (src/quant.c:55-85). */
int qmh_quantize_rows_q8(const float *x, void *y, int64_t rows, int64_t n, void *stream);
int qmh_quantize_rows_q4(const float *x, void *y, int64_t rows, int64_t n, void *stream);
/* one row of any dtype -> n floats. qm_row_to_f32 (src/quant.c:96-101) */
int qmh_row_to_f32(int dtype, const void *row, float *y, int64_t n, void *stream);

/* A weight matrix resident on the device, repacked from the reference's row layout
 * (qm_tensor rows of qm_row_bytes, src/ops.h:8-22) into the tile layout the matvec reads. */
typedef struct qmh_weight qmh_weight;
/* host_rows: rows x cols in the .qlm / qm_tensor layout. NULL on error. */
qmh_weight *qmh_weight_upload(int dtype, int64_t rows, int64_t cols, const void *host_rows);
void qmh_weight_free(qmh_weight *w);

/* y[rows] = W x. For quantized W, x is quantized to Q8_0 first and, if xq is not NULL, the
 * quantized blocks are also written there (reference layout). qm_matvec (src/ops.c:57-61)
 * with the per-row dot_f32 / dot_q8 / dot_q4 of src/kernels_scalar.c:6-34. */
int qmh_matvec(const qmh_weight *W, const float *x, float *y, void *xq, void *stream);
/* y = W * rmsnorm(x, norm_w, eps) in one launch: the reference's qm_rmsnorm followed by
 * qm_matvec on its output (src/model.c:165-168,182-183), the fused kernel the model runs.
 * xq as for qmh_matvec (the quantized normalised activation). */
int qmh_rmsnorm_matvec(const qmh_weight *W, const float *x, const float *norm_w, float eps, float *y, void *xq,
                       void *stream);

/* C[M,N] = A[M,K] B[N,K]^T, all row-major contiguous f32. qm_matmul_nt (src/ops.c:81-90) ->
 * gemm_nt (src/gemm_driver.h:7-28), scalar-ISA rounding order (K panels of 256). */
int qmh_matmul_nt(const float *A, const float *B, float *C, int64_t M, int64_t N, int64_t K, void *stream);

/* elementwise ops of src/ops.c:93-133 (in-place where the reference is in place) */
int qmh_rmsnorm(float *out, const float *x, const float *w, int64_t n, float eps, void *stream);
int qmh_softmax(float *x, int64_t n, void *stream);
int qmh_rope(float *v, int64_t n_heads, int64_t head_dim, int64_t pos, float theta, void *stream);
int qmh_swiglu(float *gate, const float *up, int64_t n, void *stream);
/* *out = first index of the maximum. qm_argmax (src/sampler.c:27-32) */
int qmh_argmax(const float *x, int32_t n, int32_t *out, void *stream);

/* ------------------------------------------------------------------ several continuations of one prompt
 * Op level, device pointers, as above: asynchronous on the stream (NULL = the library's), 0 or -1 with a
 * message, nothing allocated. No reference counterpart (the reference runs one sequence), so these are not
 * under the bitwise contract: sums and softmax statistics are held in 32 bits (64 where a choice hangs on
 * them), results are rounded once to their type, and are the same from run to run. A step of a
 * program that answers one prompt with several sequences: qmh_paged_append the new tokens,
 * qmh_paged_attention in each layer, then for a beam search qmh_beam_select and one of the reorders.
 * The calling thread's current device must be the library's. Calls that share a workspace must not overlap;
 * graphs that may run at the same time need workspaces of their own. */

/* Keys and values in pages on the device: k and v are [n_pages][n_kv_heads][page_size][head_dim] of dtype
 * (QMH_F32, QMH_F16 or QMH_BF16), 16-byte aligned; page_size a power of two in [16, 1024], head_dim a
 * multiple of 8 in [8, 256]. A table row of page numbers says where a sequence's positions lie: position
 * t is row t % page_size of page table[t / page_size]. Tables are whole arrays, [rows][stride]; entries
 * behind a sequence's last page may hold anything (qmh_paged_attention may read those up to max_len or max_prefix, no op
 * follows them). A page number outside [0, n_pages) is never followed (each op says what it does instead). */
typedef struct {
    int32_t dtype;
    int32_t n_kv_heads, head_dim, page_size;
    int64_t n_pages;
    void *k, *v;
} qmh_pages;

/* The rotation of queries and keys: pairs of the first rot_dim elements of a head are turned by
 * position * f_i radians, i < rot_dim / 2, and scaled by magnitude; the others stay. f_i = theta^(-2i / rot_dim),
 * stretched for contexts longer than first_len by `scaling`:
 *   QMH_ROTARY_LINEAR  f_i / factor
 *   QMH_ROTARY_NTK     theta * factor^(rot_dim / (rot_dim - 2)) in theta's place (rot_dim > 2)
 *   QMH_ROTARY_BANDS   f_i (w + (1 - w) / factor), w = (first_len f_i / 2 pi - low) / (high - low) held to [0, 1]: pairs
 *                      that turn more than `high` times in first_len positions stay, fewer than `low` are slowed
 *   QMH_ROTARY_YARN    the same with the ramp over pair numbers: w = 1 - (i - a) / (b - a) held to [0, 1], where
 *                      c(n) = rot_dim ln(first_len / (2 pi n)) / (2 ln theta), a = max(floor c(high), 0),
 *                      b = min(ceil c(low), rot_dim - 1), b - a at least 0.001
 * Pairs are (2i, 2i + 1) (QMH_ROTARY_PAIRS, as qmh_rope) or (i, i + rot_dim / 2) (QMH_ROTARY_HALVES).
 * Angles, their sines and cosines are computed in 64 bits for every position below max_pos (at most 2^24). */
enum { QMH_ROTARY_PAIRS = 0, QMH_ROTARY_HALVES = 1 };
enum { QMH_ROTARY_PLAIN = 0, QMH_ROTARY_LINEAR = 1, QMH_ROTARY_NTK = 2, QMH_ROTARY_BANDS = 3, QMH_ROTARY_YARN = 4 };
typedef struct {
    int32_t rot_dim, layout, scaling, max_pos, first_len;
    float theta, factor, low, high, magnitude;
} qmh_rotary_config;
typedef struct qmh_rotary qmh_rotary;
/* Tables of the rotation on the device (max_pos / 1024 + 1024 rows of rot_dim / 2 sine and cosine pairs in 64 bits).
 * Synchronous. NULL on error. Free it when no call that uses it is under way. */
qmh_rotary *qmh_rotary_create(const qmh_rotary_config *cfg);
void qmh_rotary_free(qmh_rotary *r);

/* New tokens into a paged cache, in one pass: queries and keys of each head normed (optional) and rotated
 * (optional), keys and values written to the pages, queries to q_out. Rows are of the pages' dtype.
 * Token t < n_tokens (at most 2^24) belongs to sequence seq[t] (a row of table [n_seq][table_stride]), is its position slot[t]
 * in the pages, and is rotated by position pos[t] (NULL: slot[t]; they differ where a shared prefix lies before
 * the sequence's own pages). With gains: x_i g_i / sqrt(mean x^2 + eps) over a head, g of head_dim floats.
 * q: row t at q + t * q_stride elements, n_heads heads after one another; q_out alike (q_out = q with the same
 * stride is allowed); both NULL: no queries. k, v: n_kv_heads heads a row; both NULL: queries only, and then
 * pages->k, v, table, seq and (with pos) slot are not looked at. k, v and q may be parts of the same rows.
 * A token whose seq, slot, page or pos is outside its range (slot < table_stride * page_size, pos < the rotary's
 * max_pos; pos at least 0 also without a rotation) is left out, nothing of it is written: pos or slot -1 pads a batch. No two tokens of a call may name
 * the same slot of the same sequence (the slot then holds a mixture of theirs). */
typedef struct {
    const qmh_pages *pages;
    const qmh_rotary *rotary; /* NULL: no rotation */
    int32_t n_tokens, n_heads;
    const void *q;
    int64_t q_stride;
    void *q_out;
    int64_t q_out_stride;
    const void *k;
    int64_t k_stride;
    const void *v;
    int64_t v_stride;
    const float *q_gain, *k_gain; /* NULL: no norm */
    float eps;
    int32_t n_seq;
    const int32_t *table;
    int32_t table_stride;
    const int32_t *seq, *slot, *pos;
} qmh_append_args;
int qmh_paged_append(const qmh_append_args *a, void *stream);

/* Attention of n_seq sequences with q_len queries each, over a prefix that a group's sequences share and
 * over each one's own pages: out = softmax(scale q k) v. Sequence i is in group i / (n_seq / n_groups) (n_groups divides n_seq). Its queries see
 * the group's prefix, prefix_len[g] positions in the pages of prefix_table[g] [n_groups][prefix_stride], then its own
 * pages, len[i] positions in table[i] [n_seq][table_stride]: the queries are the last q_len of these, query j
 * sees positions below len[i] - q_len + 1 + j. The prefix's keys and values are read for all queries of a
 * group together. Rows of q and out are of the pages' dtype: query j of sequence i is row i * q_len + j, n_heads
 * heads after one another (n_heads a multiple of n_kv_heads: consecutive heads share a kv head); out must not
 * overlap q. Lengths are read on the device; max_len and max_prefix are their upper bounds, from which the work
 * is divided (0: no own pages / no prefix, the table and lengths then unused).
 * Scores are held in 32 bits: products that pass their range are infinite. With 16-bit rows each position's
 * probability is rounded to their type before its product with the values, and the sum of probabilities is of the
 * rounded ones (f16: multiples of 2^-31 of the largest, so one below 2^-32 of it counts as 0); with f32 rows it is
 * not. A query that sees nothing (or only scores of -inf) gives zeros. Where a sequence's len is outside [0,
 * max_len] all its rows are NaN, where a page is outside the pool the rows of every query that sees a position of
 * it (and maybe of its earlier queries); a group's prefix does so for all its sequences. What lies in pages behind
 * a length has no effect, whatever it holds. A position below len is the sequence's: an infinite or NaN value
 * there may reach its queries that do not see it, too.
 * scale: any sign, at most 2^127 in magnitude.
 * ws: qmh_paged_attention_ws(a) bytes (0 for bad arguments), 16-byte aligned, any contents. */
typedef struct {
    const qmh_pages *pages;
    int32_t n_heads, n_seq, q_len, n_groups;
    const void *q;
    int64_t q_stride;
    void *out;
    int64_t out_stride;
    const int32_t *table, *len;
    int32_t table_stride, max_len;
    const int32_t *prefix_table, *prefix_len;
    int32_t prefix_stride, max_prefix;
    float scale;
} qmh_attention_args;
size_t qmh_paged_attention_ws(const qmh_attention_args *a);
int qmh_paged_attention(const qmh_attention_args *a, void *ws, size_t ws_bytes, void *stream);

/* A beam search's choice: the n_out best continuations of each group of n_beams rows of logits. Row b of a group
 * continues with token t at score[b] + logits[b][t] - log sum exp logits[b], in 64 bits; the best come first,
 * among equals the lower beam, then the lower token. logits: row r = group * n_beams + b at logits + r * stride
 * elements of dtype (QMH_F32, QMH_F16, QMH_BF16), read as aligned 16 bytes: up to 15 on either side of a row are
 * read, too, and have no effect. done (NULL or [rows]): a nonzero row is finished, its one continuation is token
 * eos at score[b]. Continuations at -inf or NaN are none (a row of score -inf has none: a group's first step gives
 * its other beams -inf; a row with a NaN or +inf logit has none); places that stay over get score -inf, parent -1
 * and token -1. out_*: [n_groups][n_out]; out_parent is b.
 * n_beams and n_out at most 64, vocab at most 2^24. out_score may be score where n_out = n_beams.
 * ws: qmh_beam_select_ws(a) bytes (0 for bad arguments), 16-byte aligned, any contents. */
typedef struct {
    int32_t dtype, n_groups, n_beams, vocab, n_out, eos;
    const void *logits;
    int64_t stride;
    const float *score;
    const int32_t *done;
    float *out_score;
    int32_t *out_parent, *out_token;
} qmh_beam_args;
size_t qmh_beam_select_ws(const qmh_beam_args *a);
int qmh_beam_select(const qmh_beam_args *a, void *ws, size_t ws_bytes, void *stream);

/* The states of surviving beams: dst's sequence j of each group takes src's sequence parent[j] of that group
 * (parent [n_groups][n_beams] on the device, as qmh_beam_select gives them; outside [0, n_beams): its own).
 * State of sequence i = group * n_beams + j: n_outer x n_rows pieces of `live` bytes, at outer_stride * o + seq_stride * i +
 * row_stride * r; bytes between the pieces stay as they are. dst = src moves in place (any parents); otherwise
 * the two must not overlap, nor may the pieces among themselves. n_beams at most 64. */
typedef struct {
    int64_t n_outer, outer_stride, seq_stride, n_rows, row_stride, live;
} qmh_beam_state;
int qmh_beam_reorder(const qmh_beam_state *s, void *dst, const void *src, const int32_t *parent, int32_t n_groups,
                     int32_t n_beams, void *stream);
/* The same for sequences' own pages, in place: positions below len[parent] of the parent's pages go to the
 * same positions of the sequence's own (table [n_groups * n_beams][table_stride], len on the device, at most
 * max_len, a longer one counts as max_len, one below 0 as 0). Tables and lengths stay (beams of a group are usually equally long; a
 * program that keeps them otherwise reorders len with qmh_beam_reorder). A page outside the pool is neither read nor written.
 * No page may be in two rows of a group's tables. */
int qmh_paged_reorder(const qmh_pages *pages, const int32_t *table, int32_t table_stride, const int32_t *len,
                      int32_t max_len, const int32_t *parent, int32_t n_groups, int32_t n_beams, void *stream);

/* ------------------------------------------------------------------ model level (host arguments) */

/* qm_config (src/model.h:8-11) */
typedef struct {
    int32_t dim, hidden_dim, n_layers, n_heads, n_kv_heads, vocab_size, max_seq;
    float rope_theta, norm_eps;
} qmh_config;

/* A host tensor as the reference's qm_tensor describes it (src/ops.h:9-15): dtype, shape
 * (ne[0] outermost) and a pointer to rows of qm_row_bytes. */
typedef struct {
    int32_t dtype;
    int32_t ndim;
    int64_t ne[4];
    const void *data;
} qmh_tensor_view;

typedef struct qmh_model qmh_model;

/* Build the device model from host tensors the caller already holds (the reference's
 * qm_model after qm_model_load, src/model.c:35-117). layers[9*l + k] is layer l's
 * {attn_norm, wq, wk, wv, wo, ffn_norm, w1, w2, w3}[k] (src/model.h:13-15). Shapes are
 * validated as src/model.c:20-32,48-77 do. cfg->max_seq sizes the KV cache. NULL on error. */
qmh_model *qmh_model_create(const qmh_config *cfg, const qmh_tensor_view *tok_embd, const qmh_tensor_view *norm,
                            const qmh_tensor_view *output, const qmh_tensor_view *layers);
/* Open a .qlm file (format of src/qlm_file.h:1-9) and create the device model from it.
 * max_seq <= 0 keeps the file's context, else caps it (src/model.c:53). NULL on error. */
qmh_model *qmh_model_load(const char *path, int32_t max_seq);
void qmh_model_free(qmh_model *m);
const qmh_config *qmh_model_config(const qmh_model *m);
/* The configuration a .qlm file gives the model, read and validated as qm_model_load does
 * before it touches tensors (src/model.c:35-53: the seven u32 keys, rope_theta / norm_eps with
 * their defaults, the head checks, the max_seq cap; the first entry of a duplicated key wins, as
 * qlm_find_kv's does, src/qlm_file.c:181-185). Needs no device. 0, or -1 with a message. */
int qmh_qlm_config(const char *path, int32_t max_seq, qmh_config *out);

/* One token at position pos; returns model-owned logits[vocab] in pinned host memory, or
 * NULL for token outside [0, vocab) or pos outside [0, max_seq). qm_model_forward
 * (src/model.c:158-191). */
float *qmh_model_forward(qmh_model *m, int32_t token, int32_t pos);

/* n tokens at positions pos0..pos0+n-1, enqueued as one batch with no host round trip between
 * positions. KV cache contents and logits are bitwise those of n sequential qmh_model_forward
 * calls (the reference's prompt loop, src/main.c:127-130). logits: NULL, or host memory for
 * n*vocab floats. 0 or -1. */
int qmh_model_prefill(qmh_model *m, const int32_t *tokens, int32_t n, int32_t pos0, float *logits);

/* Greedy decode on the device: n_steps forwards starting with token at pos, each next token
 * the first argmax of the previous logits (reference bench/bench.c:143-149). out[k], k < n_steps,
 * receives the argmax of the logits of the forward at position pos+k (the token fed at pos+k+1).
 * No host round trip between steps. */
int qmh_model_greedy(qmh_model *m, int32_t token, int32_t pos, int32_t n_steps, int32_t *out);

/* ------------------------------------------------------------------ batched decode (bs > 1) */

/* n_seq independent sequences decoded together over one model's weights (no reference counterpart:
 * the reference decodes one sequence, src/model.c:158-191). Each sequence has its own KV cache of
 * the model's max_seq positions, separate from the model's own. Per sequence, logits and KV contents
 * are bitwise those of the single-sequence qmh_model_forward at the same tokens and positions.
 * Needs quantized weights and head_dim <= 128, a multiple of 4; n_seq in [1, min(max_seq, 512)]. NULL on error. */
typedef struct qmh_batch qmh_batch;
qmh_batch *qmh_batch_create(qmh_model *m, int32_t n_seq);
void qmh_batch_free(qmh_batch *b);
/* One step: sequence i takes tokens[i] at position pos[i] (any mix of positions). logits: NULL, or
 * host memory for n_seq x vocab floats. Synchronous. 0 or -1. */
int qmh_batch_forward(qmh_batch *b, const int32_t *tokens, const int32_t *pos, float *logits);
/* n_steps greedy steps of every sequence on the device, from tokens[i] at pos[i]: out[k*n_seq + i]
 * is sequence i's argmax after step k (the token it takes at step k+1). ms (optional): device time
 * of the n_steps steps from HIP events. 0 or -1. */
int qmh_batch_greedy(qmh_batch *b, const int32_t *tokens, const int32_t *pos, int32_t n_steps, int32_t *out,
                     double *ms);

/* Beam search state: sequence j of each group of n_beams (which divides n_seq) takes the first n_pos positions
 * of the KV cache of sequence parent[j] of its group (host array [n_seq]; outside [0, n_beams): its own), in
 * place, all layers. Synchronous. 0 or -1. */
int qmh_batch_reorder(qmh_batch *b, const int32_t *parent, int32_t n_beams, int32_t n_pos);
/* Beam search on the device: the batch's sequences are groups of n_beams (at most 64; it divides n_seq). Every
 * sequence of group g holds the same prompt (positions below pos[g]); the search starts with tokens[g] at pos[g] and
 * makes n_steps steps, each the forward of every sequence (logits bitwise those of qmh_batch_forward), then the
 * n_beams best continuations of the group (qmh_beam_select: sums of log probabilities in 64 bits, each step's rounded to
 * float), their caches reordered. A hypothesis that took eos (-1: none) is finished: it keeps its score and repeats
 * eos. out[i * n_steps + k]: token k of hypothesis i, best first within a group (-1 throughout where the vocabulary
 * leaves fewer than n_beams); scores[i] its sum (-inf there). The caches end as the hypotheses' own, at pos[g] + n_steps.
 * ms (optional): device time of the steps. No host round trip between steps. 0 or -1. */
int qmh_batch_beam(qmh_batch *b, int32_t n_beams, const int32_t *tokens, const int32_t *pos, int32_t n_steps, int32_t eos,
                   int32_t *out, float *scores, double *ms);

/* ------------------------------------------------------------------ sampler */

/* qm_sampler (src/sampler.h:8-16): temperature / top-k / top-p sampling with an xorshift64*
 * stream. Results are token for token and rng state for rng state those of the reference's
 * qm_sample on the same logits (its float and double roundings included). */
typedef struct qmh_sampler qmh_sampler;

/* qm_sampler_init (src/sampler.c:6-16): the same normalisation (temperature < 0 -> 0, top_k < 0
 * -> 0, top_p outside (0, 1] -> 1, seed 0 -> 0x9e3779b97f4a7c15); device scratch replaces the
 * arena arrays. n_vocab in [1, 2^24]. NULL on error. */
qmh_sampler *qmh_sampler_create(int32_t n_vocab, float temperature, int top_k, float top_p, uint64_t seed);
void qmh_sampler_free(qmh_sampler *s);
/* qm_sample (src/sampler.c:50-106) of device logits[n_vocab]: the token is written to device
 * memory *out, asynchronously on the stream. Greedy configurations (temperature 0 or top_k 1)
 * take the first argmax and leave the rng alone, as the reference does. */
int qmh_sample(qmh_sampler *s, const float *logits, int32_t *out, void *stream);
/* qmh_sample on the library stream, synchronously: the token, or -1 on error. */
int32_t qmh_sample_sync(qmh_sampler *s, const float *logits);
/* The rng state (qm_sampler.rng) after the library stream's work. */
int qmh_sampler_rng(const qmh_sampler *s, uint64_t *state);
/* Diagnostics of the last non-greedy draw (no reference counterpart): diag[0] the serial double
 * sum of the exponentials, [1] 0 when every chunk certificate held, else nonzero: the sums were
 * then recomputed by one serial pass (as they are for every draw of a sampler created while the
 * environment variable QMH_SAMPLER_SERIAL is set), so the token stays exact, [2] chunks replayed serially
 * for that sum, [3] candidates, [4] k, [5] nucleus size m, [6] chunks replayed for the nucleus
 * sum, [7] nucleus mass. probs (NULL or host [n_vocab]): the normalised probabilities. */
int qmh_sampler_diag(const qmh_sampler *s, double diag[8], float *probs);

/* qmh_sample without a sampler object, allocating nothing: no counterpart in the reference. It is
 * for callers that cannot allocate device memory (code under HIP graph capture, serving loops).
 * The same draw as qmh_sample with a sampler created by qmh_sampler_create from these parameters;
 * *rng (device memory) holds the xorshift64* state and is advanced in place,
 * *out (device) receives the token, asynchronously on the stream (NULL = the library's). Scratch:
 * one static device array of 3186944 bytes per GPU, held until the process ends, so n_vocab is at
 * most 131072 (-1 otherwise). Calls that overlap on one GPU race on that array. qmh_init must have
 * run. 0 or -1. */
int qmh_sample_noalloc(const float *logits, int32_t n_vocab, float temperature, int top_k, float top_p,
                       uint64_t *rng, int32_t *out, void *stream);

/* Sampled decode on the device: n_steps forwards starting with token at pos, each next token
 * qm_sample of the previous logits (the generation loop of src/main.c:131-141). out[k] receives
 * the token sampled from the logits at position pos+k. No host round trip between steps. EOS does
 * not stop the loop (the reference stops there: cut out[] at the first EOS for its output). */
int qmh_model_sample(qmh_model *m, qmh_sampler *s, int32_t token, int32_t pos, int32_t n_steps, int32_t *out);

/* ------------------------------------------------------------------ measurement
 * No reference counterpart (the reference times with a host clock, bench/bench.c:11-38).
 * Stages of one decode step: 0 = fused RMSNorm+QKV matvec (+RoPE, KV write), 1 = Wo matvec
 * (+residual), 2 = fused RMSNorm+W1|W3 matvec (+SwiGLU), 3 = W2 matvec (+residual), 4 = final
 * RMSNorm+output matvec, 5 = attention scores, 6 = softmax + attention-weighted V sum, 7 = the
 * whole attention in one launch (scores, softmax and V sum; what decode steps use for positions below
 * 640, and below 1024 for head_dim 64 and 128, when the model's head shape allows it; an error for
 * other models and positions). */

/* Average device time of `iters` back-to-back launches of one stage at position pos (token 0),
 * from HIP events on the library stream; launch i uses layer i % n_layers, so weight reads come
 * from HBM rather than a cache. bytes_per_launch: weight bytes one launch streams (0 for
 * attention). Overwrites the KV cache entries at pos. */
int qmh_model_time_stage(qmh_model *m, int which, int32_t pos, int iters, double *ms_per_launch,
                         double *bytes_per_launch);
/* The reference bench's kernel rows (bench/bench.c:63-123, which time qm_matvec and qm_matmul_nt with
 * a host clock) on the device: the average device time (HIP events on the library stream) of `iters`
 * back-to-back qmh_matvec calls, call i on W[i % nw] (weights of one dtype and shape: several
 * copies make the reads come from HBM rather than a cache), and of qmh_matmul_nt calls. 0 or -1. */
int qmh_time_matvec(const qmh_weight *const *W, int nw, const float *x, float *y, int iters, double *ms_per_call);
int qmh_time_matmul_nt(const float *A, const float *B, float *C, int64_t M, int64_t N, int64_t K, int iters,
                       double *ms_per_call);
/* qmh_model_greedy, with HIP events around the n_steps graph replays (*ms = their total). */
int qmh_model_time_greedy(qmh_model *m, int32_t token, int32_t pos, int32_t n_steps, int32_t *out, double *ms);
/* qmh_model_prefill of n tokens at pos0, with HIP events around it (*ms). logits: 0 none, 1 the last
 * position's, 2 every position's (the reference's prompt loop computes them all: src/main.c:127-130);
 * they stay in device memory. */
int qmh_model_time_prefill(qmh_model *m, const int32_t *tokens, int32_t n, int32_t pos0, int logits, double *ms);
/* The reference bench's decode loop (bench/bench.c:143-149) on this model: n_steps of
 * token = argmax(qmh_model_forward(token, pos + k)), the argmax on the host over the returned (copied)
 * logits; *ms from a host clock; out (optional) receives the tokens. */
int qmh_model_time_forward(qmh_model *m, int32_t token, int32_t pos, int32_t n_steps, int32_t *out, double *ms);

/* ------------------------------------------------------------------ synthetic models */

/* Write a random-init .qlm (format src/qlm_file.h:1-9, tensor order of the reference's
 * writer): every 2-D tensor ~ N(0, 0.02) from a counter-based generator keyed by (seed,
 * tensor, element) and stored as wtype; norm gains 1.0. Results do not depend on n_threads.
 * 0 or -1. No reference counterpart in C (the reference's generator is its Python tooling). */
int qmh_gen_qlm(const char *path, const qmh_config *cfg, int wtype, uint64_t seed, int n_threads);
/* The f32 values (before quantization) of elements [k0, k0+n) of tensor number tensor_index
 * (its position in the file's tensor table) of a model written by qmh_gen_qlm with `seed`;
 * lets a checker re-quantize them with another quantizer. */
void qmh_gen_values(uint64_t seed, int tensor_index, int64_t k0, int64_t n, float *out);

#ifdef __cplusplus
}
#endif
#endif
