/*
 * qd_operators.h -- operators on the caller's device memory.
 *
 * The pieces of a beam search over a paged key-value cache, for programs that
 * hold their own tensors on the GPU: rows take over the pages of their
 * parents (qd_pages_fork), the rows of new tokens are rotated and written into
 * pages (qd_paged_append), one new token per row attends over its pages
 * (qd_paged_attention), and the best continuations are chosen from logits and
 * scores (qd_beam_select). qd_generate_beams (qwen_decode.h) runs a whole
 * search of an engine's model through them. Beside them: several drafted tokens
 * per row at once (qd_tree_attention, qd_tree_accept, qd_tree_commit), and
 * attention over a part of a long cache (qd_page_bounds, qd_sparse_attention).
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
  QD_PAGED_EXHAUSTED = 16,  /* fewer free pages than a fork needs */
  QD_TREE_BAD_PARENT = 32,  /* a node's parent that is not an earlier node */
  QD_TREE_BAD_PATH = 64     /* a path that is not of ascending nodes, or a count past them */
};

/* ---- workspace --------------------------------------------------------------
 * Device memory that attention, fork, select and accept keep partial results in. Its
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

/* ---- trees of drafted tokens ---------------------------------------------------------
 * A cheap model proposes several continuations of each row at once, as a tree of up to
 * 64 nodes: node 0 is the row's newest token, which stands; the others are proposals,
 * each the continuation of its parent. parents[r][i] is the node before node i, below i,
 * or -1: only what the cache holds comes before it. Less than -1: there is no node i
 * (rows with fewer nodes than the call; node 0 too in rows that only fill the batch).
 * The nodes' keys and values stand in the cache at the last `nodes` positions of the row,
 * in their order: node i at length - nodes + i (qd_paged_append_at). */

/* qd_paged_append with a place of its own for each token: token t is rotated for
 * positions[t] and written to position slots[t] of its row (both plus position_bias;
 * slots NULL: qd_paged_append). A drafted token is rotated for its depth in the tree and
 * stands at its node's place. A token is skipped if either is negative; a (row, slot) given
 * twice is as a (row, position) there. */
QD_API qd_status qd_paged_append_at(const qd_paged_cache *cache, const qd_append_args *args, const int32_t *slots,
                                    void *stream);

/* Attention of the nodes of a tree in each row of the cache, cache->lengths counting
 * them: node i attends to the positions before the tree, to the nodes above it and to
 * itself,
 *   out[r][i][h] = sum_j softmax_j(scale q[r][i][h] . K_j) V_j,
 * each position read once for up to 128 (FP32: 64) pairs of a node and a query head of one
 * KV head. Precision is qd_paged_attention's, but that a weight in FP16 is off by 2^-22 of
 * it or 2^-39 of the row's largest. Nodes that are not there get zeros, and so do rows of length 0, whose
 * parents are not looked at. K and V of nodes that are not seen may hold anything,
 * also values that are not finite: outputs that see such a V become NaN or infinite. A row of another length
 * gets NaN if it has a bad page, a bad parent, or a length below `nodes` or past its
 * table. q and out are [rows][nodes][heads][head_dim] with strides that are
 * multiples of 16 bytes; out may be q itself, with its strides. */
typedef struct qd_tree_attention_args {
  const void *q;
  void *out;
  int64_t q_stride;      /* from row to row */
  int64_t q_node_stride;
  int64_t q_head_stride;
  int64_t out_stride;
  int64_t out_node_stride;
  int64_t out_head_stride;
  const int32_t *parents; /* [rows][nodes] */
  uint32_t nodes;        /* up to 64 */
  uint32_t heads;        /* a multiple of kv_heads */
  float scale;
} qd_tree_attention_args;
QD_API qd_status qd_tree_attention(const qd_paged_cache *cache, const qd_tree_attention_args *args,
                                   qd_workspace *workspace, void *stream);
/* Bytes of workspace that caches of up to `rows` rows and trees of up to `nodes` need. */
QD_API qd_status qd_tree_attention_workspace(uint32_t rows, uint32_t nodes, uint32_t heads, uint32_t kv_heads,
                                             uint32_t head_dim, size_t *bytes);

/* Which drafted tokens stand: from node 0 on, the token that follows a node is picked from
 * its logits, and if a child of the node carries it (the lowest such child), the walk goes
 * on there. The token picked at the walk's last node is new.
 *   path[r][..]     the walk's nodes, -1 behind them
 *   counts[r]       how many they are, node 0 among them
 *   next_tokens[r]  the new token
 * Picked is the token of the largest logit, the lowest of equal ones; NaN counts as -inf.
 * With draws (numbers u from 0 up to 1), the least token t with
 *   sum_{i <= t} p_i > u sum_i p_i,  p_i = exp(logits[i] / temperature)
 * (in FP32, a p_i of 2^-d of the largest off by at most (1.8 d + 4) 2^-24 of itself and sums of
 * up to 8 of them by 3 x 2^-24; sums beyond in 64 bits), so that the tokens that come out are
 * distributed as the model's own. A draw below 0 or NaN
 * counts as 0, one of 1 or more picks the last token that has a probability, which -inf and
 * NaN have not; a p_i below 2^-126 of the largest may count as none. Where the largest logit
 * is past 1e30 either way, the token of the largest logit is picked. A row whose node 0 is
 * not there gets count 0 and -1, and so does one with a bad parent. The results must not
 * overlap each other or what is read, but that next_tokens may be the tokens of trees of
 * one node. */
typedef struct qd_accept_args {
  const void *logits;      /* [rows][nodes][vocab] */
  int64_t row_stride;
  int64_t node_stride;
  const int32_t *tokens;   /* [rows][nodes] what each node carries */
  const int32_t *parents;  /* [rows][nodes] */
  const float *draws;      /* [rows][nodes], or NULL */
  int32_t *path;           /* [rows][nodes] */
  int32_t *counts;         /* [rows] */
  int32_t *next_tokens;    /* [rows] */
  uint32_t *errors;        /* one word, or NULL */
  float temperature;       /* read with draws: from 1e-6 to 1e6 */
  uint32_t dtype;          /* of the logits */
  uint32_t rows;
  uint32_t nodes;          /* up to 64 */
  uint32_t vocab;          /* up to 2^24 */
  int32_t device;
} qd_accept_args;
QD_API qd_status qd_tree_accept(const qd_accept_args *args, qd_workspace *workspace, void *stream);
/* Bytes of workspace that calls of up to so many rows and nodes need. */
QD_API qd_status qd_tree_accept_workspace(uint32_t rows, uint32_t nodes, uint32_t vocab, size_t *bytes);

/* One memory that holds something of each position: `pieces` pieces (heads) of
 * piece_bytes bytes, piece n of position j of page p at
 * base + plane * plane_stride + p * page_stride + j * token_stride + n * piece_stride
 * in each of `planes` planes (layers). All in bytes. */
typedef struct qd_token_memory {
  void *base;
  int64_t plane_stride;
  int64_t page_stride;
  int64_t token_stride;
  int64_t piece_stride;
  uint32_t piece_bytes;  /* a multiple of 16, as the address and the strides are */
  uint32_t pieces;
  uint32_t planes;
  uint32_t reserved;
} qd_token_memory;

/* Moves what stands of each row's tree together: what the memories hold at node
 * path[r][i]'s position goes to position length - nodes + i, i < counts[r], as if all
 * were read before any is written. lengths_out[r] = lengths[r] - nodes + counts[r]; 0 for
 * a row of length 0, whose path is not read. Positions behind are left as they are. A row
 * with a bad length (not 0 and below `nodes`, or past the table), count, path (its nodes
 * ascend) or page moves nothing and hands its length on. Rows whose trees lie in the same
 * pages must not be committed in one call, nor memories that overlap; lengths_out must
 * not overlap lengths, counts, path or table. */
typedef struct qd_commit_args {
  const int32_t *table;
  const int32_t *lengths;
  const int32_t *path;     /* [rows][nodes] */
  const int32_t *counts;
  int32_t *lengths_out;
  int64_t table_stride;
  uint32_t *errors;        /* one word, or NULL */
  const qd_token_memory *memories; /* host array, up to 4 */
  uint32_t memory_count;
  uint32_t rows;           /* up to 65535 */
  uint32_t nodes;          /* up to 64 */
  uint32_t table_width;
  uint32_t pages;
  uint32_t page_size;      /* positions; a power of two from 16 to 1024 */
  int32_t device;
} qd_commit_args;
QD_API qd_status qd_tree_commit(const qd_commit_args *args, void *stream);

/* ---- attention over chosen pages --------------------------------------------------------
 * A row's query reads the pages whose keys may matter most to it, by bounds that are kept
 * of each page's keys: bounds[page][kv_head][0][d] is the least and [1][d] the largest value
 * of element d of the keys in the page (cache dtype, contiguous). */

/* The bounds of every page that holds one of a row's last `recent` positions, over all of
 * the row's positions in it. NaN counts as neither; a page of NaN alone gets +inf and -inf.
 * Rows that share a page write the same bounds if they hold equally much of it, else each
 * value is one of theirs. A row with a bad length or page sets an error bit; its other pages are done. */
QD_API qd_status qd_page_bounds(const qd_paged_cache *cache, void *bounds, uint32_t recent, void *stream);

/* qd_paged_attention over up to `budget` pages of each row and KV head. Of a row of n
 * pages, the first `first` and the last `last` are always read; if n > budget, of those
 * between the ones that score highest, the lower of equal ones:
 *   score(page) = sum over the KV head's query heads and d of
 *                 max(q_d low_d, q_d high_d),
 * as much as the products of the page's keys can sum to, in 64 bits. Bounds are as
 * qd_page_bounds makes them. A term with a product that is NaN (of 0 and an infinite bound,
 * of a query that is NaN) is NaN, and a score that is NaN counts as +inf.
 *   chosen[r][kv_head][..]  the columns of the table that were read, ascending, -1 behind
 *                           them (NULL: not told; not over the table or the lengths)
 * A row of n <= budget pages reads all of them. A row with a bad length gets NaN, one
 * with a bad page at least where its page is chosen, as it then is. */
typedef struct qd_sparse_args {
  const void *q;
  void *out;
  int64_t q_stride;
  int64_t q_head_stride;
  int64_t out_stride;
  int64_t out_head_stride;
  const void *bounds;  /* [pages][kv_heads][2][head_dim] */
  int32_t *chosen;     /* [rows][kv_heads][budget], or NULL */
  uint32_t heads;
  uint32_t budget;     /* at least first + last, and 1 */
  uint32_t first;
  uint32_t last;       /* at least 1 */
  float scale;
} qd_sparse_args;
QD_API qd_status qd_sparse_attention(const qd_paged_cache *cache, const qd_sparse_args *args, qd_workspace *workspace,
                                     void *stream);
/* Bytes of workspace that calls of up to so many rows, columns of the table and pages need. */
QD_API qd_status qd_sparse_attention_workspace(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                               uint32_t table_width, uint32_t budget, size_t *bytes);

#ifdef __cplusplus
}
#endif

#endif /* QD_QD_OPERATORS_H_ */
