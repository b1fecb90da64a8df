/* si_paged.h - C ABI of the paged key-value cache of the B200 decode backend.
 *
 * Operators for many sequences over one pool of cache pages: rotary positions
 * and the append of new keys and values, attention of one new token a
 * sequence, eviction by accumulated attention weight, and the verification of
 * drafted tokens by probabilities. si_cuda.h has their single-sequence
 * counterparts (si_rope, si_attention_decode, si_model_verify_many, si_argmax)
 * and the conventions, which hold here too:
 *  - every function returns SI_OK or a negative SI_E_*; the text is in
 *    si_last_error(ctx), or si_global_last_error() when ctx is NULL;
 *  - `_dev` functions take device pointers, enqueue their work on `stream`
 *    (cudaStream_t as void*, NULL = the context's stream) and return without
 *    synchronising; nothing is allocated. They may be captured into a CUDA
 *    graph and replayed;
 *  - all descriptions are host structs, read before the call returns.
 * The arguments are checked before the context is looked at, so a call with
 * ctx = NULL checks a description without a device.
 *
 * The reference has one contiguous f32 cache per layer (cache.rs:1-171) and
 * no counterpart of these operators.
 *
 * Errors found on the device (a page number outside the pool, a length beyond
 * the page table or the weights' rows, a drafted token outside the vocabulary)
 * neither read nor write out of bounds: the offending token is left out, and
 * si_ctx_synchronize or a host-memory call of the context returns SI_E_INVALID
 * for it, once: the first that finds it, at the latest the first that follows
 * the work's end.
 *
 * Calls that overlap on the GPU need workspaces of their own, and so do CUDA
 * graphs that may be replayed at the same time.
 */
#ifndef SI_PAGED_H
#define SI_PAGED_H

#include "si_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations and caches (SI_CACHE_F32 / SI_CACHE_BF16 and
 * IEEE half). */
#define SI_ELEM_F32 0u
#define SI_ELEM_BF16 1u
#define SI_ELEM_F16 2u

/* A paged cache: element (page, head, token of the page, dim) of either pool
 * lies at page * page_stride + head * head_stride + token * token_stride +
 * dim (elements), so any order of pages, heads and tokens is described by the
 * strides. Slot t of sequence b is token t % page_tokens of page
 * pages[b * pages_stride + t / page_tokens]. Entries of the page table that no
 * slot in use needs are not read as pages. Rows of the batch may share pages
 * as long as no operator writes them; pools that are written have every
 * (page, head, token) in a place of its own. */
typedef struct si_paged_kv {
  void* k;                  /* pools, 16-byte aligned */
  void* v;
  const int32_t* pages;     /* [sequences][pages_stride] */
  uint64_t num_pages;       /* pages of a pool, below 2^31 */
  uint64_t page_stride, head_stride, token_stride; /* multiples of 8 */
  uint64_t pages_stride;    /* at least max_pages */
  uint32_t elem;            /* SI_ELEM_BF16 or SI_ELEM_F16 */
  uint32_t kv_heads, head_dim; /* head_dim: a multiple of 8, at most 256 */
  uint32_t page_tokens;     /* any number from 1 */
  uint32_t sequences;       /* at most 4096 */
  uint32_t max_pages;       /* page_tokens * max_pages below 2^31 */
} si_paged_kv;
/* Host only: where slot `slot` of a sequence whose page is `page` lies in a
 * pool (elements). SI_E_INVALID for a page, head or slot out of range. */
int si_paged_kv_offset(const si_paged_kv* kv, int64_t page, uint64_t slot, uint32_t head, uint64_t* offset);

/* ---- rotary positions and append ----------------------------------------- */
#define SI_ROPE_INTERLEAVED 0u /* pairs (2i, 2i + 1), as si_rope */
#define SI_ROPE_HALF 1u        /* pairs (i, i + rotary_dim / 2) */
/* Scaling of the positions for contexts longer than the model was trained on;
 * f_i = theta^(-2i / rotary_dim) is the frequency of pair i:
 *   NONE    f_i
 *   LINEAR  f_i / factor
 *   NTK     theta * factor^(rotary_dim / (rotary_dim - 2)) in place of theta
 *           (rotary_dim 2: theta)
 *   YARN    f_i / factor (1 - k) + f_i k, k falling from 1 to 0 between the
 *           pairs that turn beta_fast and beta_slow times over `original`
 *           positions; rotated values times 0.1 ln(factor) + 1
 *   BANDED  f_i where a pair turns at least `high` times over `original`
 *           positions, f_i / factor below `low` times, linear in the number of
 *           turns between */
#define SI_ROPE_SCALE_NONE 0u
#define SI_ROPE_SCALE_LINEAR 1u
#define SI_ROPE_SCALE_NTK 2u
#define SI_ROPE_SCALE_YARN 3u
#define SI_ROPE_SCALE_BANDED 4u
typedef struct si_rope_scaling {
  uint32_t kind;
  double factor;               /* all but NONE; at least 1 */
  double original;             /* YARN, BANDED: positions of the training */
  double beta_fast, beta_slow; /* YARN: beta_fast > beta_slow > 0 */
  double low, high;            /* BANDED: high > low > 0 */
} si_rope_scaling;
/* Host only: the frequencies as turns (2 pi radians) a position in units of
 * 2^-64, [rotary_dim / 2], and the factor on rotated values. `scaling` NULL:
 * NONE. position * turn in 64-bit integers is the pair's angle modulo one
 * turn, off by the table's own rounding only: at most |position| * 2^-65
 * turns. The caller copies the table to the device. */
int si_rope_table(double theta, uint32_t rotary_dim, const si_rope_scaling* scaling, uint64_t* turns, float* scale);

/* For every token t: queries rotated into q_out; keys rotated and values as
 * they are, rounded to the cache's type, written to slot slot[t] of sequence
 * sequence[t]. A token whose slot is negative is padding: nothing of it is
 * written, neither cache nor q_out. Two tokens of a call must not share a
 * (sequence, slot). q and q_out may be the same memory with the same strides;
 * otherwise no element of q_out is one of q, k or v, nor are its rows each
 * other's. Strides count elements; dims are contiguous.
 * With weights and positions, the arrays that attention adds to and eviction
 * reads, every appended slot starts with weight 0 and its token's position in
 * each kv head. A slot behind a cut holds what the token that left it had
 * gathered, so a cache that is evicted from needs this with every append. */
typedef struct si_paged_append {
  const void* q;            /* [tokens][query_heads][head_dim]; NULL: none */
  void* q_out;
  const void* k;            /* [tokens][kv_heads][head_dim]; k and v NULL: queries only */
  const void* v;
  uint64_t q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
  uint64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  const int32_t* sequence;  /* [tokens]; NULL: token t belongs to sequence t */
  const int32_t* slot;      /* [tokens] */
  const int32_t* position;  /* [tokens]; NULL: the slot */
  const uint64_t* rope;     /* device copy of si_rope_table's turns; NULL only with rotary_dim 0 */
  float rope_scale;
  uint32_t elem;            /* type of q, k, v and q_out: SI_ELEM_* */
  uint32_t tokens;          /* 0: nothing to do */
  uint32_t query_heads, rotary_dim, rope_layout;
  float* weights;           /* [sequences][kv_heads][weights_stride]; NULL: not wanted. Needs k and v */
  int32_t* positions;       /* the same */
  uint64_t weights_stride;  /* of both, entries; a slot at or beyond it is out of range */
} si_paged_append;
int si_paged_append_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_append* a, void* stream);

/* ---- attention of one new token a sequence -------------------------------- */
/* out[b][i] = sum over t < lengths[b] of softmax_t(scale q[b][i] . k_t) v_t,
 * query head i reading kv head i / (query_heads / kv_heads); the new token's
 * own key and value are in the cache already (si_paged_append_dev). A sequence
 * of length 0 gets zeros (and lse = -inf): rows of a padded batch have length
 * 0. Cached values at slots in use are taken to be finite; whatever lies in
 * other slots is not read. Sums and the softmax are held in f32. With f32
 * queries and output the products keep 24 bits of queries and probabilities
 * over a bf16 cache and 22 bits over an f16 cache; with queries of the cache's
 * own 16-bit type, probabilities keep 16 bits (bf16) or 22 (f16). The same
 * call gives the same bits; how the sums group depends on all lengths of the
 * batch.
 * With weights_out, weights_out[b][h][t] = weights_in[b][h][t] + the sum of
 * the probabilities of slot t over the query heads of kv head h, for
 * t < lengths[b]; other entries are left as they are. weights_in may be
 * weights_out (otherwise they share nothing), or NULL for zeros. */
typedef struct si_paged_attention {
  const void* q;            /* [sequences][query_heads][head_dim] */
  void* out;                /* no element of q: several blocks read a query; rows apart from each other */
  uint64_t q_seq_stride, q_head_stride, out_seq_stride, out_head_stride;
  const int32_t* lengths;   /* [sequences], each at most max_pages * page_tokens */
  float scale;              /* 0: 1 / sqrt(head_dim) */
  uint32_t elem;            /* type of q and out: SI_ELEM_* */
  uint32_t query_heads;     /* a multiple of kv_heads */
  float* lse;               /* [sequences][query_heads] natural log of the sum of exp(score); NULL: not wanted */
  const float* weights_in;  /* [sequences][kv_heads][weights_stride] */
  float* weights_out;       /* NULL: no weights */
  uint64_t weights_stride;  /* at least the longest length */
  void* work;               /* 16-byte aligned */
  uint64_t work_bytes;
} si_paged_attention;
/* Host only: bytes of workspace a call needs (with or without weights). With
 * weights every score is kept between two kernels: sequences * kv_heads *
 * max_pages * page_tokens * (group of query heads, rounded up to even) * 4
 * bytes, by the room of the page table, not by the lengths or the pool. 64
 * sequences with tables for 131,072 slots, 8 kv heads and groups of 4 need
 * 1.07 GB. */
int si_paged_attention_workspace(const si_paged_kv* kv, uint32_t query_heads, int weights, uint64_t* bytes);
int si_paged_attention_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_attention* a, void* stream);

/* ---- eviction by accumulated weight ---------------------------------------- */
/* Cuts every sequence longer than `budget` tokens to `budget`, each kv head by
 * itself. A token stays if its position is below `sink` or among the last
 * `recent` before next_position[b]; of the others those with the smallest
 * weight leave, of equal ones the lowest slot first (NaN counts as smaller
 * than any number). Kept tokens of slots >= budget move into the slots that
 * became free below it, both in order; nothing else moves. Attention does not
 * depend on the order of slots: keys carry their position, and from the first
 * cut on a slot's number is not its token's position any more: positions and
 * next_position are then needed, and every append has to start its slots'
 * weights and positions anew (si_paged_append). The pages that hold
 * no slot below the new length can be given to other sequences afterwards.
 * Should more than `budget` tokens be protected (positions that repeat),
 * the protected ones of the lowest slots leave, after all others.
 * Entries of weights_out and positions_out at slots below the new length are
 * written, others left as they are. Each `_in` may be its `_out`; otherwise
 * inputs and outputs share nothing. Launches are planned for the most slots
 * that the page table and weights_stride have room for (lengths are on the
 * device): tables much wider than the rows cost time. */
typedef struct si_paged_evict {
  const int32_t* lengths_in;    /* [sequences] */
  int32_t* lengths_out;         /* min(length, budget) */
  const float* weights_in;      /* [sequences][kv_heads][weights_stride] */
  float* weights_out;
  const int32_t* positions_in;  /* as weights_in; NULL: slot t holds position t */
  int32_t* positions_out;       /* NULL: not wanted */
  const int32_t* next_position; /* [sequences]; NULL: lengths_in. Not lengths_out, unless all three are one */
  uint64_t weights_stride;      /* of all four, entries; at least the longest length */
  uint32_t budget;              /* at least 1 */
  uint32_t sink, recent;        /* sink + recent <= budget */
  void* work;                   /* 16-byte aligned */
  uint64_t work_bytes;
} si_paged_evict;
/* Host only. SI_E_UNSUPPORTED beyond 393216 slots a sequence. */
int si_paged_evict_workspace(const si_paged_kv* kv, uint64_t* bytes);
int si_paged_evict_dev(si_ctx* ctx, const si_paged_kv* kv, const si_paged_evict* a, void* stream);

/* ---- verification of drafted tokens ---------------------------------------- */
/* Speculative sampling: draft i of sequence b (token x) is accepted while
 * uniform[b][i] * draft[b][i][x] < target[b][i][x]. The token after the
 * accepted ones is drawn from max(target - draft, 0) of the first rejected
 * place, or from the target's row after the last draft when all are accepted:
 * the lowest token whose cumulative weight exceeds last_uniform[b] times the
 * total. Acceptance is exact, and sums are held in 64 bits. The same call gives
 * the same token; in a batch of another size a row's sums are taken in another
 * order, which moves a border by about 1e-16 of the total and so the token
 * about once in 10^10 draws. Negative, infinite and NaN entries count as 0. If
 * the difference is 0 everywhere the target's row itself is drawn from; if that
 * is too, next = -1. draft NULL: the drafter has no probabilities (1 for its
 * token): x is accepted with probability target[x], and the difference is the
 * target's row without x. A drafted token outside the vocabulary is rejected
 * and reported. */
typedef struct si_verify_drafts {
  const float* target;      /* [sequences][drafts + 1][vocab] probabilities */
  const float* draft;       /* [sequences][drafts][vocab], or NULL */
  uint64_t target_seq_stride, target_row_stride, draft_seq_stride, draft_row_stride;
  const int32_t* tokens;    /* [sequences][drafts] */
  const int32_t* counts;    /* [sequences] drafts of each sequence, at most `drafts`; NULL: all */
  const float* uniform;     /* [sequences][drafts] in [0, 1) */
  const float* last_uniform;/* [sequences] in [0, 1) */
  int32_t* accepted;        /* [sequences]; may be counts */
  int32_t* next;            /* [sequences]; not accepted */
  uint32_t sequences;       /* at most 65535 */
  uint32_t drafts;          /* 0..32 */
  uint32_t vocab;           /* below 2^31 */
  void* work;               /* 16-byte aligned */
  uint64_t work_bytes;
} si_verify_drafts;
/* Host only. 16 bytes for any call; the operator keeps nothing in them. */
int si_verify_drafts_workspace(uint32_t sequences, uint32_t vocab, uint64_t* bytes);
int si_verify_drafts_dev(si_ctx* ctx, const si_verify_drafts* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SI_PAGED_H */
