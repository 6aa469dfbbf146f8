/*
 * qd_operators.h -- operators on the caller's device memory.
 *
 * The pieces of a beam search over a paged key-value cache, for programs that
 * hold their own tensors on the GPU: rows take over the pages of their
 * parents (qd_pages_fork), the rows of new tokens are rotated and written into
 * pages (qd_paged_append), one new token per row attends over its pages
 * (qd_paged_attention), and the best continuations are chosen from logits and
 * scores (qd_beam_select). qd_generate_beams (qwen_decode.h) runs a whole
 * search of an engine's model through them.
 *
 * Conventions:
 *   - pointers are device memory unless they say host; sizes and strides are
 *     in elements unless they say bytes; the innermost dimension (head_dim, a
 *     row's columns) is contiguous;
 *   - a call checks its arguments on the host and queues kernels on `stream`
 *     (a hipStream_t; NULL is the null stream), which belongs to `device`. It
 *     makes that device current while it queues and puts the caller's back. It
 *     does not wait, allocate or copy to the host, and may be captured into a
 *     HIP graph;
 *   - what stands in device memory (lengths, page ids, positions, parents) is
 *     checked by the kernels: nothing out of range is read or written. What is
 *     wrong there sets a bit of *errors (a zeroed uint32_t, or NULL) and has
 *     the effect that the call names;
 *   - tensors must not overlap unless a call says so;
 *   - calls return qd_status; qd_last_error() has the text.
 *
 * No counterpart in the reference, which decodes one sequence greedily over a
 * contiguous cache (examples/qwen/README.md:431-432).
 */
#ifndef QD_QD_OPERATORS_H_
#define QD_QD_OPERATORS_H_

#include <stddef.h>
#include <stdint.h>

#include "qd/qwen_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of the `errors` words. */
enum {
  QD_PAGED_BAD_LENGTH = 1,  /* a length below 0 or past the table's columns */
  QD_PAGED_BAD_PAGE = 2,    /* a page id that is needed and not in [0, pages) */
  QD_PAGED_BAD_POSITION = 4,/* a position past the table's columns or the rotary tables */
  QD_PAGED_BAD_ROW = 8,     /* a row or parent that does not exist */
  QD_PAGED_EXHAUSTED = 16   /* fewer free pages than a fork needs */
};

/* ---- workspace --------------------------------------------------------------
 * Device memory that attention, fork and select keep partial results in. Its
 * owner allocates one of the largest size its calls ask for and may pass it to
 * any of them, but to one call at a time: calls on the same stream, or graphs
 * replayed on the same stream, follow each other; work that may run at the same
 * time (two streams, two graphs on two streams) needs a workspace each. The sizes
 * that are asked for serve smaller calls too, as each says. Destroying one waits
 * for the device. */
typedef struct qd_workspace qd_workspace;
QD_API qd_status qd_workspace_create(int32_t device, size_t bytes, qd_workspace **workspace);
QD_API qd_status qd_workspace_destroy(qd_workspace *workspace);

/* ---- paged key-value cache ----------------------------------------------------
 * K and V of `pages` pages of `page_size` positions. Position p of cache row r
 * is token p % page_size of page table[r * table_stride + p / page_size]; its
 * head h starts at element page * page_stride + token * token_stride +
 * h * head_stride of k and of v. Rows may share pages. */
typedef struct qd_paged_cache {
  void *k;
  void *v;
  int64_t page_stride;
  int64_t token_stride;    /* at least head_dim */
  int64_t head_stride;     /* at least head_dim; strides and addresses are multiples of 16 bytes */
  const int32_t *table;    /* [rows][table_width] */
  int64_t table_stride;
  const int32_t *lengths;  /* [rows] valid positions of each row */
  uint32_t *errors;        /* one word, or NULL */
  uint32_t rows;
  uint32_t table_width;
  uint32_t pages;
  uint32_t page_size;      /* a power of two from 16 to 1024 */
  uint32_t kv_heads;
  uint32_t head_dim;       /* 64 or 128 */
  uint32_t dtype;          /* qd_dtype of K and V and of the queries and outputs beside them */
  int32_t device;
} qd_paged_cache;

/* Fills host tables cos and sin [positions][rotary_dim / 2] for
 * qd_paged_append: cos(p f_i) and sin(p f_i), f_i = theta^(-2 i / rotary_dim),
 * angles in 64 bits, rounded once. stretch > 1 scales the positions for a
 * context that many times longer than `original` positions: frequencies that
 * turn more than `fast` times (32) within `original` positions stay, those that
 * turn less than `slow` times (1) are divided by stretch, those between are
 * mixed by the logarithm of their turns (which are not rounded to whole dimensions
 * first); both tables are multiplied by 0.1 ln(stretch) + 1. qd_paged_append takes
 * any tables: a checkpoint trained with other angles brings its own. Host only. */
QD_API qd_status qd_rope_table(double theta, uint32_t rotary_dim, uint32_t positions, double stretch,
                               uint32_t original, double fast, double slow, float *cos_table, float *sin_table);

/* Writes `tokens` new tokens: token t belongs to cache row rows[t] (NULL: row
 * t) at position positions[t] + position_bias. Its query heads are rotated
 * into q_out, its key heads rotated and its value heads copied into the page
 * of that position. The rotation takes the first rotary_dim of head_dim
 * elements, in pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where
 * `interleaved` is nonzero: (a, b) -> (a c - b s, b c + a s) with c and s from
 * row `position` of cos_table and sin_table [table_positions][rotary_dim / 2],
 * in FP32, rounded once. rotary_dim 0: nothing is rotated and the tables may be
 * NULL. q NULL: keys and values only. q_out may be q itself, with its stride. A
 * token whose position is negative is skipped: nothing of it is read or written. A
 * (row, position) given twice gets one token's row or the other's, not
 * necessarily of one whole token. cache->lengths is not read. A token whose row,
 * position or page does not exist is not written, and its q_out row is NaN. */
typedef struct qd_append_args {
  const void *q;        /* [tokens][heads][head_dim], or NULL */
  const void *k;        /* [tokens][kv_heads][head_dim] */
  const void *v;
  void *q_out;
  int64_t q_stride;     /* from token to token; heads are head_dim apart; multiples of 16 bytes */
  int64_t k_stride;
  int64_t v_stride;
  int64_t q_out_stride;
  const int32_t *positions;
  const int32_t *rows;
  int32_t position_bias;
  uint32_t tokens;
  uint32_t heads;
  uint32_t rotary_dim;  /* a multiple of 8, at most head_dim */
  uint32_t interleaved;
  uint32_t table_positions;
  const float *cos_table;
  const float *sin_table;
} qd_append_args;
QD_API qd_status qd_paged_append(const qd_paged_cache *cache, const qd_append_args *args, void *stream);

/* Attention of one new token per cache row: query head h of row r over
 * positions 0 .. lengths[r] - 1 of KV head h / (heads / kv_heads),
 *   out[r][h] = sum_j softmax_j(scale q[r][h] . K_j) V_j,
 * statistics and sums in FP32 (products are summed before they are divided, by
 * weights up to 2^8: finite for |V| below 2^89). 16-bit types multiply a weight
 * as two numbers, off by at most 2^-16 of it in BF16, and in FP16 by 2^-22 of it
 * or 2^-51 of the row's largest, whichever is more; an infinite V makes the
 * outputs that it reaches infinite or NaN. A row of length 0 gets zeros; what the
 * pages hold past a row's length is not read. A row with a bad length or page
 * gets NaN. q and out are [rows][heads][head_dim] with strides that are multiples
 * of 16 bytes; out may be q itself, with its strides. The result of a row does not
 * depend on when its parts finish (they are joined in order), but how its
 * positions are split goes by all rows' lengths and by how many positions tables
 * and pages can hold, as the lengths are not known when the call queues. A page
 * that several rows list is read for each of them. */
typedef struct qd_attention_args {
  const void *q;
  void *out;
  int64_t q_stride;      /* from row to row */
  int64_t q_head_stride;
  int64_t out_stride;
  int64_t out_head_stride;
  uint32_t heads;        /* a multiple of kv_heads */
  float scale;
} qd_attention_args;
QD_API qd_status qd_paged_attention(const qd_paged_cache *cache, const qd_attention_args *args, qd_workspace *workspace,
                                    void *stream);
/* Bytes of workspace that caches of up to `rows` rows need with these heads. */
QD_API qd_status qd_paged_attention_workspace(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                              size_t *bytes);

/* ---- pages: fork, copy on write, grow, free ------------------------------------
 * refs[p] counts who holds page p: each table row that lists it, and whoever
 * else the caller counts; 0 is free. A page consists of `plane_count` pieces:
 * piece n of page p is `bytes` bytes at base + n * plane_stride +
 * p * page_stride, for each of the listed memories (K and V, all layers). */
typedef struct qd_page_memory {
  void *base;
  int64_t plane_stride;  /* bytes */
  int64_t page_stride;   /* bytes, at least `bytes` */
  uint64_t bytes;        /* a multiple of 16, as the address and the strides are */
  uint32_t planes;
  uint32_t reserved;
} qd_page_memory;

/* One step of every row: row r of the new table takes over row parents[r] of
 * the old one (NULL: its own; -1: none, the row is released) with the pages that
 * hold the parent's `length` positions, and gets room for `append` more:
 *   - refs follow: a page is held by as many rows as list it; entries of an old
 *     row behind its length are released too;
 *   - if append > 0 and the length ends inside a page that others hold too, the
 *     row gets a fresh page with a copy of that one's content. Where only rows
 *     of this table hold it, all as the page that they go on in, the lowest of
 *     them keeps it;
 *   - further fresh pages cover length + append. Fresh pages are the free ones
 *     of the lowest ids, dealt to the rows in order, a copy before new pages.
 * table_out gets the ids and -1 behind them, lengths_out the lengths plus
 * append (0 for a released row). An old row is contiguous: its ids end at its
 * first negative entry or at the last column. Nothing happens by halves: with a
 * bad length, parent or page, a row that grows past the table's columns
 * (QD_PAGED_BAD_LENGTH) or too few free pages, an error bit is set and table,
 * lengths and refs are handed on as they were, with no page copied. (The rows then
 * have no room for new tokens: an append that is queued behind such a fork, at the
 * last positions of lengths_out, writes over what stands there.) table_out and
 * lengths_out must not overlap table and lengths: a program keeps two of each and
 * takes them in turn. Forks that share refs follow each other, as calls
 * that share a workspace do. */
typedef struct qd_fork_args {
  const int32_t *table;   /* [rows][table_width] */
  const int32_t *lengths;
  const int32_t *parents;
  int32_t *table_out;
  int32_t *lengths_out;
  int32_t *refs;          /* [pages], in place */
  int64_t table_stride;
  int64_t table_out_stride;
  uint32_t *errors;       /* one word, or NULL */
  const qd_page_memory *memories; /* host array, up to 4 */
  uint32_t memory_count;
  uint32_t rows;          /* up to 1024 */
  uint32_t table_width;
  uint32_t pages;
  uint32_t page_size;     /* positions; a power of two from 16 to 1024 */
  uint32_t append;
  int32_t device;
} qd_fork_args;
QD_API qd_status qd_pages_fork(const qd_fork_args *args, qd_workspace *workspace, void *stream);
/* Bytes of workspace that forks of up to so many rows and pages need. */
QD_API qd_status qd_pages_fork_workspace(uint32_t rows, uint32_t pages, size_t *bytes);

/* ---- beam selection --------------------------------------------------------------
 * Of each group's beams x vocab continuations the best k. Continuation (b, t)
 * scores
 *   scores[b] + log softmax(logits[b])[t],
 * sums in 64 bits (exponentials and 16 of them FP32), candidates compared in 64 bits. Higher
 * scores come first; continuations of one beam go by their logits, then by the
 * lower token; equal scores of two beams by the lower beam. NaN counts as -inf.
 * A beam whose score is not finite has no continuation; one that is done (done[b]
 * nonzero) has one, the token `eos`, at no cost. Where fewer than k
 * continuations have a finite score, the rest of the places go, at -inf, to the
 * others in order of beam and token.
 *   scores_out[g][i]   FP32
 *   parents[g][i]      g * beams + b: the row the i-th goes on from
 *   tokens[g][i]       t
 *   done_out[g][i]     1 if that beam was done or t is eos (NULL with done NULL)
 * The results must not be the tensors that are read: a program keeps two of
 * scores and done and takes them in turn. */
typedef struct qd_select_args {
  const void *logits;    /* [groups][beams][vocab] */
  int64_t group_stride;
  int64_t beam_stride;   /* not negative; 0: all beams read the same row */
  const float *scores;   /* [groups][beams] */
  const uint8_t *done;   /* [groups][beams], or NULL */
  float *scores_out;     /* [groups][k] */
  int32_t *parents;
  int32_t *tokens;
  uint8_t *done_out;
  uint32_t dtype;        /* of the logits */
  uint32_t groups;
  uint32_t beams;        /* up to 32 */
  uint32_t vocab;        /* up to 2^24 */
  uint32_t k;            /* up to 64 and beams x vocab */
  uint32_t eos;          /* read with done */
  int32_t device;
} qd_select_args;
QD_API qd_status qd_beam_select(const qd_select_args *args, qd_workspace *workspace, void *stream);
/* Bytes of workspace that calls of up to so many groups, beams, places and tokens need. */
QD_API qd_status qd_beam_select_workspace(uint32_t groups, uint32_t beams, uint32_t k, uint32_t vocab, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* QD_QD_OPERATORS_H_ */
