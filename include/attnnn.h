/* attnnn.h -- C ABI of libattnnn.so, the gfx950 (MI355X) implementation of the
 * autoregressive token loop of attention_nn (sample.py running model.py).
 *
 * Plain C: pointers, sizes, ints.  No torch or C++ types cross this boundary.
 * Every entry point returns ANN_OK (0) or a negative ANN_E_* code; the message
 * of the last failure on the calling thread is ann_last_error().  Arguments
 * are validated on the host before any kernel is launched.
 *
 * Ownership: the caller allocates every device buffer (weights, KV cache,
 * workspace, inputs, outputs) and keeps it alive while a context uses it; the
 * library keeps raw pointers and never frees them.  A context owns host state
 * only.  One context per stream; calls on one context are not thread-safe.
 * Work is enqueued on the caller's hipStream_t (passed as void*); calls return
 * without synchronising unless noted.
 *
 * Reference interfaces replaced (henneberger/attention_nn):
 *   ann_create / ann_pack_weights / ann_bind  <- GPT(cfg) + params dict
 *                                                (model.py:138-153, sample.py:31-38)
 *   ann_forward_logits                        <- GPT.logits (model.py:223-263)
 *   ann_forward_loss                          <- GPT.__call__ (model.py:180-221) with the
 *                                                fused softcap CE (softcap_ce, model.py:
 *                                                121-132; ce_softcap_fwd, metal_kernels.py:
 *                                                153-193, 213-221)
 *   ann_prefill / ann_decode_step             <- the per-token loop body
 *                                                (sample.py:42-50: logits of the
 *                                                last row, /temp, top-k, categorical)
 *   ann_op_relu2                              <- relu2 (metal_kernels.py:37-47,62-68)
 *   ann_op_rope_ht                            <- rope_ht (metal_kernels.py:87-134)
 *   ann_op_rope_tables                        <- make_rope_tables (metal_kernels.py:144-150)
 *   ann_op_rms_norm                           <- rms (model.py:48-49)
 *   ann_op_adam_step                          <- adam_step (metal_kernels.py:241-270)
 *   ann_op_muon_momentum                      <- muon_momentum (metal_kernels.py:277-300)
 *   ann_op_muon_apply                         <- muon_apply (metal_kernels.py:306-329)
 *   ann_op_polar_express(_ws_bytes)           <- polar_express (muon.py:28-44)
 *   ann_op_normuon(_ws_bytes)                 <- normuon_rescale (muon.py:47-63)
 *   ann_op_qk_norm_rope(_bwd)                 <- rms and rope_ht of q and k, and their
 *                                                gradient (model.py:244-247)
 *   ann_op_paged_*                               no counterpart: attention over a cache
 *                                                (model.py:248-254) that sequences of
 *                                                any lengths share, and their tables
 *   ann_op_sample_logits                      <- /temp, top-k and categorical of given
 *                                                logits (sample.py:45-49), with top_p, min_p
 */
#ifndef ATTNNN_H
#define ATTNNN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ANN_OK 0
#define ANN_E_ARG (-1)      /* bad argument, shape or size */
#define ANN_E_STATE (-2)    /* call out of order (e.g. decode before prefill) */
#define ANN_E_CAPACITY (-3) /* batch / context / buffer exceeds what was bound */
#define ANN_E_HIP (-4)      /* a HIP runtime call failed */

#define ANN_MAX_LONG_LAYERS 8
#define ANN_DTYPE_F32 0
#define ANN_DTYPE_BF16 1

/* GPTConfig (model.py:30-45) plus the capacities the caller will bind. */
typedef struct ann_config {
  int32_t d;          /* model_dim */
  int32_t L;          /* num_layers */
  int32_t H;          /* num_heads; head_dim = d / H */
  int32_t V;          /* vocab_size (rows of embed / columns of lm_head) */
  int32_t V_sample;   /* rows sampling considers (50257, sample.py:45) */
  int32_t window;     /* sliding window of the short layers */
  int32_t n_long;     /* number of full-causal layers */
  int32_t long_layers[ANN_MAX_LONG_LAYERS];
  float attn_scale;   /* 0.1 */
  float rope_base;    /* 1024 */
  float rms_eps;      /* 1e-6 */
  int32_t max_batch;  /* sequences per call */
  int32_t max_ctx;    /* KV-cache length per sequence; also RoPE table length */
  int32_t max_tokens; /* rows per forward call (B*T of the largest prefill) */
} ann_config;

/* Device pointers to the reference fp32 parameter dict (model.py:52-77). */
typedef struct ann_params_f32 {
  const float* embed;         /* (V, d) */
  const float* lm_head;       /* (d, V) */
  const float* attn_bank;     /* (L, 4, d, d): q, k, v, o, each (in, out) */
  const float* fc_bank;       /* (L, d, 4d) */
  const float* proj_bank;     /* (L, 4d, d) */
  const float* resid_lambdas; /* (L, 2) */
  const float* post_lambdas;  /* (L, 2) */
  const float* x0_lambdas;    /* (L,) */
  const float* sa_lambdas;    /* (L, 2) */
} ann_params_f32;

/* Sampling of one step (sample.py:45-49).  temperature == 0 selects greedy
 * (argmax over the first V_sample logits, lowest index on ties).  top_k <= 0
 * or >= V_sample keeps every row.  Draws use Philox4x32-10 with counter
 * (step, row) and key seed. */
typedef struct ann_sampling {
  float temperature;
  int32_t top_k;
  uint64_t seed;
  uint64_t step;
} ann_sampling;

typedef struct ann_ctx ann_ctx;

const char* ann_last_error(void);
int ann_version(void);

/* Validate cfg and create a context (host state only). */
int ann_create(const ann_config* cfg, ann_ctx** out);
void ann_destroy(ann_ctx* ctx);

/* Bytes the caller must allocate for each device buffer. */
size_t ann_weight_bytes(const ann_config* cfg);
size_t ann_kv_bytes(const ann_config* cfg);
size_t ann_workspace_bytes(const ann_config* cfg);

/* Convert the fp32 parameter dict (device pointers) into the packed bf16
 * layout in wbuf (ann_weight_bytes bytes): bf16 casts, sa_lambdas folded into
 * the QKV / O weights with the two roundings of model.py:239-241, every
 * matrix stored (out, in) so a row of the output is a contiguous dot product,
 * RoPE tables appended.  Enqueued on stream. */
int ann_pack_weights(ann_ctx* ctx, const ann_params_f32* src, void* wbuf,
                     size_t wbytes, void* stream);

/* Attach the caller's buffers; sizes are checked against the ann_*_bytes. */
int ann_bind(ann_ctx* ctx, void* wbuf, size_t wbytes, void* kv, size_t kvbytes,
             void* workspace, size_t wsbytes);

/* Forget all sequences (the next call must be a prefill). */
int ann_reset(ann_ctx* ctx);

/* GPT.logits: tokens (B, T) int32 at positions 0..T-1 -> softcapped fp32
 * logits (B, T, V).  Leaves the KV cache filled for those B sequences, so
 * ann_decode_step may follow. */
int ann_forward_logits(ann_ctx* ctx, const int32_t* tokens, int32_t B, int32_t T,
                       float* logits, void* stream);

/* GPT.__call__ (training forward, loss only): tokens and targets (B, T) int32
 * on the device, positions 0..T-1.  Writes the mean over the B*T rows of
 * log(sum_v exp(zc[v])) - zc[target], zc = 23*sigmoid((z + 5)/7.5) and
 * z = bf16(rms(x) @ lm_head) over all V columns, as one fp32 to *loss, and the
 * per-row losses (B*T fp32) to row_loss when non-null.  The logits never
 * reach memory.  Targets must lie in [0, V) (not checked on the device: an
 * out-of-range target leaves its row's value undefined).  Leaves the KV cache
 * filled like ann_forward_logits. */
int ann_forward_loss(ann_ctx* ctx, const int32_t* tokens, const int32_t* targets, int32_t B,
                     int32_t T, float* loss, float* row_loss, void* stream);

/* Prefill B prompts of T tokens (positions 0..T-1), then sample one token
 * per sequence into out_tok (B).  logits (B, V) of the last rows is written
 * when non-null. */
int ann_prefill(ann_ctx* ctx, const int32_t* tokens, int32_t B, int32_t T,
                const ann_sampling* s, int32_t* out_tok, float* logits,
                void* stream);

/* One decode step: tokens (B) are appended at each sequence's next position,
 * one token per sequence is sampled into out_tok (B).  out_tok may equal
 * tokens.  logits (B, V) written when non-null. */
int ann_decode_step(ann_ctx* ctx, const int32_t* tokens, int32_t B,
                    const ann_sampling* s, int32_t* out_tok, float* logits,
                    void* stream);

/* Current length of the bound sequences (host mirror; 0 after reset). */
int ann_context_length(const ann_ctx* ctx);

/* ---- operators (the reference's kernel-level API) --------------------- */

/* y = max(x, 0)^2 computed in fp32, stored in dtype; n elements. */
int ann_op_relu2(const void* x, void* y, size_t n, int32_t dtype, void* stream);

/* Half-truncated RoPE of x (B, T, H, D) in dtype: pairs (2p, 2p+1), p < D/4,
 * rotated by the angle of position pos0 + t from the fp32 tables cs, sn
 * (rows >= pos0 + T, D/4 columns); the other dims pass through.
 * inverse != 0 applies the transpose (the reference's BWD variant). */
int ann_op_rope_ht(const void* x, void* y, const float* cs, const float* sn,
                   int32_t B, int32_t T, int32_t H, int32_t D, int32_t pos0,
                   int32_t inverse, int32_t dtype, void* stream);

/* cs, sn (seq_len, head_dim/4) fp32: theta = t * (1/base)^linspace(0,1,D/4). */
int ann_op_rope_tables(float* cs, float* sn, int32_t seq_len, int32_t head_dim,
                       float base, void* stream);

/* y = x * rsqrt(mean(x^2) + eps) over rows of length dim, fp32 math. */
int ann_op_rms_norm(const void* x, void* y, int32_t rows, int32_t dim, float eps,
                    int32_t dtype, void* stream);

/* ---- measurement (no reference counterpart) ------------------------------
 * While enabled, every launch of one kernel class inside the forward calls is
 * bracketed by a HIP event pair recorded on the call's stream (up to
 * max_launches).  ann_profile_read waits for the recorded events and returns
 * the summed duration and the launch count, then clears the record.
 * kind -1 disables. */
#define ANN_PROF_LM_HEAD 0
#define ANN_PROF_QKV 1
#define ANN_PROF_O 2
#define ANN_PROF_FC 3
#define ANN_PROF_PROJ 4
#define ANN_PROF_ATTN 5
#define ANN_PROF_STEP 6   /* the persistent batch-1 decode kernel (whole step) */
int ann_profile_enable(ann_ctx* ctx, int32_t kind, int32_t max_launches);
int ann_profile_read(ann_ctx* ctx, float* total_ms, int32_t* launches);

/* ---- optimizer step (MuonAdam, muon.py:66-137) ----------------------------
 * All arrays are device fp32 unless noted; n elements; outputs may alias the
 * matching inputs.  Scalars as the reference passes them. */
/* adam_step: m' = b1 m + (1-b1) g; v' = b2 v + (1-b2) g^2;
 * u = m' / (sqrt(v') + eps) * step_size; u += p * eff_wd where u * p > 0; p' = p - u. */
int ann_op_adam_step(const float* p, const float* g, const float* m, const float* v, size_t n,
                     float beta1, float beta2, float eps, float step_size, float eff_wd,
                     float* p_out, float* m_out, float* v_out, void* stream);
/* muon_momentum: buf' = buf + (1-mu)(g - buf); geff = g + mu (buf' - g). */
int ann_op_muon_momentum(const float* g, const float* buf, size_t n, float mu, float* geff,
                         float* buf_out, void* stream);
/* muon_apply: p' = p - p*wd*lr (where u*p >= 0) - u*lr. */
int ann_op_muon_apply(const float* p, const float* u, size_t n, float lr, float wd, float* p_out,
                      void* stream);
/* polar_express: g (batch, M, N) fp32 -> out (batch, M, N) bf16, M and N
 * multiples of 64; ws: ann_op_polar_express_ws_bytes(batch, M, N) bytes. */
size_t ann_op_polar_express_ws_bytes(int32_t batch, int32_t M, int32_t N);
int ann_op_polar_express(const float* g, int32_t batch, int32_t M, int32_t N, void* out,
                         void* ws, size_t ws_bytes, void* stream);
/* normuon_rescale: v (batch, M, N) bf16; second_mom (batch, M) if M >= N else
 * (batch, N), updated in place; out (batch, M, N) fp32. */
size_t ann_op_normuon_ws_bytes(int32_t batch, int32_t M, int32_t N);
int ann_op_normuon(const void* v, float* second_mom, int32_t batch, int32_t M, int32_t N,
                   float beta2, float* out, void* ws, size_t ws_bytes, void* stream);

/* normuon_rescale and muon_apply in one pass (muon.py:121-127): the rescaled
 * update u is not stored, p' = p - p*wd*lr (where u*p >= 0) - u*lr.  N a
 * multiple of 8; v, p and p_out 16-byte aligned; p_out may be p; ws:
 * ann_op_normuon_ws_bytes(batch, M, N). */
int ann_op_normuon_update(const void* v, float* second_mom, int32_t batch, int32_t M, int32_t N,
                          float beta2, const float* p, float lr, float wd, float* p_out, void* ws,
                          size_t ws_bytes, void* stream);

/* NorMuon without an allocation.  No counterpart in the reference: for
 * callers that cannot allocate device memory (code under HIP graph capture,
 * tight training or serving loops, harnesses that forbid hipMalloc).  Same
 * arguments and results as ann_op_normuon, minus the workspace: the scratch
 * is a fixed device array of ann_op_normuon_noalloc_max_bytes() (4 MiB) inside
 * the library, one per GPU, held until the process ends, so batch * max(M, N)
 * may be at most 524288 (ANN_E_CAPACITY beyond).  The function itself calls
 * no hipMalloc / hipFree.  Every call on one GPU shares that GPU's array:
 * calls that overlap on one GPU (other streams or threads) race.  The stream
 * must belong to the current device. */
size_t ann_op_normuon_noalloc_max_bytes(void);
int ann_op_normuon_noalloc(const void* v, float* second_mom, int32_t batch, int32_t M, int32_t N,
                           float beta2, float* out, void* stream);

/* ---- queries and keys ------------------------------------------------------
 * Each head's row normalised and its first half turned by the token's position
 * in one pass (model.py:244-247): n = x / sqrt(mean(x^2) + eps), pairs p < D/4
 * as in ann_op_rope_ht.  fp32 inside, rounded once to dtype. */
typedef struct ann_qk_rows {
  const void* q;         /* (B, T, Hq, D) in dtype, last dimension contiguous */
  const void* k;         /* (B, T, Hk, D); Hk may be 0 */
  const void* v;         /* ann_op_paged_append only: (B, T, Hk, D) */
  const void* gq;        /* ann_op_qk_norm_rope_bwd only: gradients of the outputs */
  const void* gk;
  void* q_out;           /* (B, T, Hq, D) contiguous */
  void* k_out;           /* (B, T, Hk, D) contiguous */
  int64_t q_stride[3];   /* elements from batch to batch, token to token, head to head */
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t gq_stride[3];
  int64_t gk_stride[3];
  const float* cs;       /* RoPE tables (table_rows, D/4) */
  const float* sn;
  const int32_t* pos;    /* null: token t is at pos0 + t */
  int32_t pos_each;      /* pos: 0 (B,), token t at pos[b] + t; 1 (B, T) */
  int32_t pos0;
  int32_t table_rows;    /* a device position outside the table takes its nearest row */
  int32_t B, T, Hq, Hk, D;
  int32_t dtype;
  float eps;
} ann_qk_rows;
int ann_op_qk_norm_rope(const ann_qk_rows* r, void* stream);
/* The gradients of q and k from those of the outputs, to q_out and k_out. */
int ann_op_qk_norm_rope_bwd(const ann_qk_rows* r, void* stream);

/* ---- paged key/value cache -----------------------------------------------
 * Sequences of any lengths share a pool of pages.  Entry e of sequence s is
 * slot e % page_size of page table[s][e / page_size].  The new tokens of a call
 * lie behind one another, those of sequence s in rows starts[s] ..
 * starts[s + 1] - 1 (starts never falls; rows from starts[seqs] on belong to no
 * sequence and are left as they were); lens[s] counts its entries with these,
 * so the last new token is entry lens[s] - 1.  table, starts and lens are
 * device arrays: ids that are no page are never written to and read page 0,
 * lengths outside the table end at it.  Rows of queries, keys, values and
 * cache slots are 16-byte aligned (strides multiples of 8, slots at most 2^25
 * elements apart).  A head of the cache serves heads / cache heads query heads
 * behind one another.  Pages that a call writes belong to one sequence, and its
 * rows share no memory (no stride of 0, k is not v); pages that are only read may be
 * shared. */
typedef struct ann_paged {
  void* k;               /* bf16, (pages, heads, page_size, head_dim) by the strides */
  void* v;
  int64_t k_page, k_head, k_slot;   /* elements */
  int64_t v_page, v_head, v_slot;
  const int32_t* table;  /* (seqs, cols), rows table_row elements apart */
  int64_t table_row;
  const int32_t* starts; /* seqs + 1 */
  const int32_t* lens;   /* seqs */
  int32_t pages, page_size;   /* page_size a power of two, 16 .. 1024 */
  int32_t heads, head_dim;    /* head_dim 64 or 128 */
  int32_t seqs, cols;         /* cols * page_size <= 2^30 */
  int32_t rows;               /* rows of new tokens */
} ann_paged;

/* Queries and keys of c->rows new tokens (r: bf16, B 1, T rows) normalised and
 * turned as above, queries to q_out, keys and values to their entries.  A
 * token's position is its entry, or pos[row] (pos_each 1). */
int ann_op_paged_append(const ann_paged* c, const ann_qk_rows* r, void* stream);

/* A new token at entry e sees the entries j <= e and, with window > 0, e - j <
 * window: out = softmax(scale q.k_j) v_j (rows, heads, head_dim) bf16, lse
 * (rows, heads) fp32 the natural log of the softmax sum, or null.  A token that
 * sees nothing gets 0 and -infinity.  q (rows, heads, head_dim) bf16 by
 * strides (q_row at most 2^25, heads * q_head at most 2^28; rows * heads at most
 * 2^30); out may be q, by contiguous rows.  ws: ann_op_paged_attention_ws_bytes
 * bytes (16-byte aligned), one for each call in flight. */
size_t ann_op_paged_attention_ws_bytes(const ann_paged* c, int32_t heads, int32_t window);
int ann_op_paged_attention(const ann_paged* c, const void* q, int64_t q_row, int64_t q_head,
                           int32_t heads, float scale, int32_t window, void* out, float* lse,
                           void* ws, size_t ws_bytes, void* stream);

/* The same where sequences begin with the same entries: groups of them, group g
 * sequences groups[g] .. groups[g + 1] - 1 (groups never falls), share the first lens[g]
 * entries of table[g] (count, cols; by rows `row` elements apart), which their own
 * tables name too (or copies of them).  A prefix is read once for its group's tokens.  Sequences of no
 * group share nothing.  ws: ann_op_paged_attention_shared_ws_bytes bytes (16-byte
 * aligned), one for each call in flight. */
typedef struct ann_paged_prefix {
  const int32_t* groups;   /* count + 1 */
  const int32_t* table;
  int64_t row;
  const int32_t* lens;     /* count */
  int32_t count, cols;     /* cols * page_size <= 2^30 */
} ann_paged_prefix;
size_t ann_op_paged_attention_shared_ws_bytes(const ann_paged* c, const ann_paged_prefix* x,
                                              int32_t heads, int32_t window);
int ann_op_paged_attention_shared(const ann_paged* c, const ann_paged_prefix* x, const void* q,
                                  int64_t q_row, int64_t q_head, int32_t heads, float scale,
                                  int32_t window, void* out, float* lse, void* ws, size_t ws_bytes,
                                  void* stream);

/* weight_out[s][j] = weight[s][j] + sum over sequence s's new tokens that see
 * entry j and over heads of exp(scale q.k_j - lse), lse as
 * ann_op_paged_attention gives it; entries behind the sequence keep their
 * weight.  weight and weight_out (seqs, cols * page_size) fp32, rows w_row and
 * out_row elements apart; they may be the same, or share nothing.  c->v is not
 * read.  The sums' order does not depend on what else runs: results are
 * reproducible.  No workspace is needed: ann_op_paged_weight_ws_bytes gives 0, and
 * ws is not read. */
size_t ann_op_paged_weight_ws_bytes(const ann_paged* c, int32_t heads);
int ann_op_paged_weight(const ann_paged* c, const void* q, int64_t q_row, int64_t q_head,
                        int32_t heads, const float* lse, float scale, int32_t window,
                        const float* weight, int64_t w_row, float* weight_out, int64_t out_row,
                        void* ws, size_t ws_bytes, void* stream);

/* Eviction by weight: a sequence of more than `keep` entries keeps its last
 * `recent` and, of the others, those of the largest weight (of equal ones the
 * lower entry; NaN below every number), min(len, keep) in all, moved in order
 * to entries 0 .. of the pages in out_table (seqs, out_cols; rows out_row
 * elements apart).  out_table is the table itself (in place: no two sequences
 * share a page) or names pages that the table does not, each once.  index (seqs,
 * keep): the entry each came from, -1 behind them; new_lens (seqs); weight_out
 * (seqs, cols * page_size): their weights, 0 behind them; it may be weight, and
 * new_lens may be c->lens.  c->starts is not read. */
int ann_op_paged_evict(const ann_paged* c, const int32_t* out_table, int64_t out_row,
                       int32_t out_cols, const float* weight, int64_t w_row, int32_t keep,
                       int32_t recent, int32_t* index, int32_t* new_lens, float* weight_out,
                       int64_t wo_row, void* stream);

/* Pages given to sequences and taken back.  refs[p] counts the tables that name
 * page p; a page is free where it is not above 0.  An id that is no page
 * (negative, or pages and more) is none.  table (seqs, cols) names each sequence's
 * pages, lens[s] counts its entries.  table_out and refs_out may be table (by the same
 * rows) and refs, else share no memory with another operand.  All device arrays. */
typedef struct ann_paged_table {
  const int32_t* table;  /* rows table_row elements apart */
  int64_t table_row;
  const int32_t* lens;
  const int32_t* refs;   /* pages */
  int32_t* table_out;
  int64_t out_row;
  int32_t* refs_out;
  int32_t pages, page_size;   /* page_size a power of two, 16 .. 1024 */
  int32_t seqs, cols;         /* cols * page_size <= 2^30 */
} ann_paged_table;

/* A step's tokens get their pages: sequence s is to grow by new_tokens[s] (below 0: 0)
 * entries, and needs a page for each column that these touch and that names none.
 * Sequences are served in order, whole or not at all: s where its entries fit its table
 * row and the rows and pages asked for by it and those before it (that fit theirs) are
 * no more than `rows` and the free pages; one that needs no page needs only the rows.  The
 * columns of those served take the free pages in ascending order (refs_out 1).
 * starts (seqs + 1) and new_lens (seqs; it may be t->lens) then describe the step as ann_paged takes
 * it, and row r of the step is entry pos[r] of sequence seq[r], slot[r] = page *
 * page_size + place in the page; -1 behind the last row (seq, pos, slot: rows).  ws:
 * ann_op_paged_assign_ws_bytes bytes (16-byte aligned), one for each call in flight. */
size_t ann_op_paged_assign_ws_bytes(const ann_paged_table* t, int32_t rows);
int ann_op_paged_assign(const ann_paged_table* t, const int32_t* new_tokens, int32_t rows,
                        int32_t* starts, int32_t* new_lens, int32_t* seq, int32_t* pos,
                        int64_t* slot, void* ws, size_t ws_bytes, void* stream);

/* Sequences cut to lens entries (0: ended) give their pages back: each column behind
 * them that names a page takes one from its count, and is -1 in table_out. */
int ann_op_paged_release(const ann_paged_table* t, void* stream);

/* ---- tokens from logits -----------------------------------------------------
 * One token of each row by given random numbers.  m is the row's largest entry; an
 * entry x weighs w = exp((x - m) / temperature) where that is at least max(min_p,
 * 2^-40), else 0 (entries equal to m: 1); of these the ones not below the k-th largest
 * entry stay, where top_k is in 1 .. cols - 1; of these, where top_p < 1, the ones not
 * below the largest t for which the entries at or above t weigh at least top_p of
 * all.  The token is the first index at which the running sum of the weights
 * passes u times their sum (u outside [0, 1): the nearest number inside); logprob
 * the log of its share.  A temperature not above 0 takes the lowest index of the
 * largest entry.  A NaN is never drawn; a row without an entry above -infinity
 * gives -1 and -infinity.  Weights are formed in 64 bits and added exactly. */
typedef struct ann_logit_rows {
  const void* logits;        /* (rows, cols) in dtype, rows `stride` elements apart */
  int64_t stride;
  const float* u;            /* rows */
  const float* temperature;  /* a setting for each row, or null: the one for all */
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all;     /* >= 0, as min_p and top_p */
  int32_t top_k_all;
  float top_p_all;
  float min_p_all;
  int32_t rows, cols;        /* cols in 1 .. 2^20 */
  int32_t dtype;
  int32_t* ids;              /* rows */
  float* logprob;            /* rows, or null */
} ann_logit_rows;
int ann_op_sample_logits(const ann_logit_rows* r, void* stream);

/* Device status of the decode steps (no reference counterpart).  The
 * cross-work-group waits of the persistent batch-1 step and of the decode
 * attention's split combine are bounded; one that gives up sets a device flag
 * and the step's output is not valid.  Synchronises `stream`, returns
 * ANN_E_HIP (and clears the flag) if it is set, else ANN_OK. */
int ann_check_device(ann_ctx* ctx, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ATTNNN_H */
