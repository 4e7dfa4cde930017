/* mechta_paged.h -- many sequences on one paged K/V cache on one MI355X, in the same library as mechta_kv.h
 * (libmechta_kv.so). Error codes are the MKV_E_* of mechta_kv.h and the message of a failed call is in
 * mkv_last_error(); a refused call changes nothing and enqueues nothing, and one that fails on its way to the device (MKV_E_HIP,
 * or MKV_E_NOMEM of the host) leaves every sequence as it was, so that it can be made again, and the batch too, unless it
 * was the copying of pages that failed: then no batch stands.
 *
 * A handle owns a pool of `pages` pages. A page holds `page` consecutive positions of one sequence, K and V of every
 * layer. Sequences are numbered 0 .. seqs - 1; a sequence is the list of its pages and a length, both kept on the host
 * and mirrored on the device. Sequences forked off one prompt share its full pages (each page counts its owners); a page
 * that is filled partly always belongs to one sequence alone.
 *
 * A step: mpg_begin names the sequences of the batch and how many new tokens each has, takes the pages they need and
 * lays out the work of every layer; then, layer by layer, mpg_append writes the new rows (rotating K, and q beside) and
 * mpg_attend attends. The tokens of a batch are packed: those of the first sequence, then those of the second, and so
 * on; rows of the arguments behind the last token are neither read nor written. A batch stands until the next mpg_begin,
 * or until pages change hands (mpg_fork, mpg_copy, mpg_free, mpg_compact, mpg_set_len, mpg_reserve): then appends and
 * attention are refused until a new mpg_begin.
 *
 * Ordering: every call is enqueued on the handle's HIP stream; none waits, except mpg_create, mpg_sync and mpg_destroy.
 * What goes up to the device (mpg_begin; the page calls that end a batch; mpg_read_rows, uncaptured, where pages are new)
 * goes through four pinned buffers: such a call waits where the stream is four of them behind, and for a larger buffer
 * when it needs one. Calls of one handle come from one thread at a time and run
 * on one stream at a time: the handle's workspaces are shared by all its calls. A call makes the handle's device
 * current while it runs.
 *
 * Graphs: mpg_append, mpg_attend and mpg_read_rows may be captured, the others are refused on a stream that is
 * capturing. What a captured call works on is read on the device when the graph runs: after another mpg_begin a replay
 * of the same graph does that batch, of any sequences, counts and lengths; tokens behind the rows that
 * were captured are left out. Replays are ordered with the handle's other calls like any call.
 *
 * Layout: per layer and K|V one array of pages, page p at p x kv_heads x page x head_dim elements. Inside a page, per kv
 * head, K is [pos/16][d/8][pos%16][8] and V [pos/32][g][d][8], where element e of group g of V is position
 * 16 (e/4) + 4 g + e%4 of its 32: the operand order of the CDNA4 16x16x32 matrix instructions, so that scores turn into
 * the weights of V without leaving their registers. mpg_read_rows gives rows [pos][kv_head][d].
 */
#ifndef MECHTA_PAGED_H
#define MECHTA_PAGED_H

#include "mechta_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mpg_store mpg_t;

/* element types: MKV_F16 (0) and MKV_F32 (1) of mechta_kv.h, and bfloat16 */
#define MPG_BF16 2

#define MPG_CTX_MAX 4194304   /* positions of a sequence at most */
#define MPG_TOKENS_MAX 262144 /* tokens of a batch at most */
#define MPG_WINDOWS_MAX 4     /* different windows of a handle's layers at most */

typedef struct mpg_config {
    int layers;
    int q_heads, kv_heads; /* q_heads a multiple of kv_heads; query head h reads kv head h / (q_heads / kv_heads) */
    int head_dim;          /* 64, 128 or 256 */
    int fmt;               /* MKV_F16 or MPG_BF16: pages, q, k, v, gate and out */
    int pages;             /* pages of the pool */
    int page;              /* positions of a page: 32, 64, 128 or 256 */
    int seqs;              /* sequences at most */
    int ctx;               /* positions of a sequence at most, <= MPG_CTX_MAX */
    int tokens;            /* tokens of a batch at most, <= MPG_TOKENS_MAX */
} mpg_config;

/* Rotary positions. dim: the rotated part of a head, even, from its first element on. layout: pairs (i, i + dim/2) or
 * (2i, 2i + 1). Pair i of position p turns by p th_i, th_i = base^(-2i/dim), scaled:
 *   MPG_LINEAR th_i / factor
 *   MPG_NTK    base taken as base factor^(dim / (dim - 2))
 *   MPG_YARN   r th_i / factor + (1 - r) th_i, r = clamp((i - lo) / max(hi - lo, 0.001), 0, 1), lo = floor(e(beta_fast)) >= 0,
 *              hi = ceil(e(beta_slow)) <= dim - 1, e(t) = dim ln(original / (2 pi t)) / (2 ln base); cos and sin times
 *              the amplitude, 0.1 ln factor + 1 (factor > 1) where it is given as 0
 *   MPG_BANDS  (1 - s) th_i / factor + s th_i, s = clamp((original th_i / (2 pi) - low) / (high - low), 0, 1)
 * Angles are computed in 64 bits and taken modulo a whole turn before cos and sin, so positions far out lose nothing. */
#define MPG_HALF 0
#define MPG_INTERLEAVED 1
#define MPG_PLAIN 0
#define MPG_LINEAR 1
#define MPG_NTK 2
#define MPG_YARN 3
#define MPG_BANDS 4
#define MPG_ROPE_DIM_MAX 512
typedef struct mpg_rope {
    int dim, layout, scaling;
    int original;                    /* the context the model was trained on (MPG_YARN, MPG_BANDS) */
    double base, factor;
    double beta_fast, beta_slow;     /* MPG_YARN: 32 and 1 */
    double low, high;                /* MPG_BANDS: 1 and 4 */
    double amplitude;                /* 0: 1, and for MPG_YARN 0.1 ln factor + 1 */
} mpg_rope;

/* What a rotation goes by, worked out once: whole turns per position of each pair, th_i / (2 pi). */
typedef struct mpg_turns {
    double turns[MPG_ROPE_DIM_MAX / 2];
    float amplitude;
    int dim, layout;
} mpg_turns;
int mpg_rope_turns(const mpg_rope* r, mpg_turns* turns);
/* th_i of the dim/2 pairs, scaled, and the amplitude (host). */
int mpg_rope_freqs(const mpg_rope* r, double* freqs, double* amplitude);
/* Rotates rows x heads vectors of dim elements at the positions pos[row] (device, int32): out = x rotated, its elements
 * behind r->dim copied. fmt: MKV_F16, MKV_F32 or MPG_BF16. x and out (device): element (row, head, d) at
 * row x *_row + head x *_head + d; out may be x with x's strides, and overlap it in no other way; the rows and heads
 * of out lie apart (strides shorter than a head, or the same for both, are refused). On the current device, enqueued on
 * `stream`. Products and sums in f32, rounded once. */
int mpg_rotate(const mpg_turns* r, int fmt, int rows, int heads, int dim, const void* x, int64_t x_row, int64_t x_head,
               const int* pos, void* out, int64_t o_row, int64_t o_head, void* stream);

/* Device bytes mpg_create allocates for the configuration (0 if it would refuse it). */
size_t mpg_bytes(const mpg_config* c);
/* Allocates the pool (zero filled), the page tables and the workspaces on the current device. windows: per layer the
 * positions a token sees, itself included (0: all before it); NULL: all 0. rope: what mpg_append rotates by, NULL: nothing.
 * stream: a hipStream_t (NULL = the default stream). */
int mpg_create(mpg_t** out, const mpg_config* c, const int* windows, const mpg_rope* rope, void* stream);
int mpg_destroy(mpg_t* h);
/* Calls from here on go to `stream`; that it comes after what the handle has on its stream before is the caller's to see to. */
int mpg_set_stream(mpg_t* h, void* stream);
int mpg_sync(mpg_t* h);

/* Length of a sequence; its pages in order (at most cap of them are written; returns how many it has, or an error);
 * pages that no sequence owns. */
int mpg_len(const mpg_t* h, int seq, int* len);
int mpg_table(const mpg_t* h, int seq, int* pages, int cap);
int mpg_free_pages(const mpg_t* h, int* n);
/* Device address of a layer's K or V pages (which = MKV_K / MKV_V), for callers that move pages themselves. */
int mpg_pages(const mpg_t* h, int layer, int which, void** base);

/* Lengthens each of n different sequences by count[i] >= 0 positions; pages are taken lowest number first, in the order
 * of the list. MKV_E_NOMEM if the pool has too few free pages, MKV_E_POS past ctx: then none is lengthened. */
int mpg_reserve(mpg_t* h, int n, const int* seq, const int* count);
/* mpg_reserve, and makes them the batch: sequence seq[i]'s last count[i] positions are its new tokens. *tokens: their
 * sum. */
int mpg_begin(mpg_t* h, int n, const int* seq, const int* count, int* tokens);
/* Shortens a sequence to len positions and gives back the pages behind them (rollback of rejected drafts). A page that
 * becomes partly filled while others own it is copied first. */
int mpg_set_len(mpg_t* h, int seq, int len);
/* Makes each empty sequence dst[i] the first len[i] positions of src[i] (len NULL: all of them). Full pages are shared,
 * a partly filled last page is copied, all layers. Destinations differ from each other and from all sources. */
int mpg_fork(mpg_t* h, int n, const int* src, const int* dst, const int* len);
/* The same with pages of its own: every page is copied. */
int mpg_copy(mpg_t* h, int n, const int* src, const int* dst);
/* Empties n different sequences; pages without owners are free again. */
int mpg_free(mpg_t* h, int n, const int* seq);
/* Moves pages so that those in use are the lowest: the lowest free page takes the lowest page behind the part in use,
 * and so on. *moved (may be NULL): how many moved. */
int mpg_compact(mpg_t* h, int* moved);

/* Writes the batch's K and V rows of one layer into its pages and, with q, rotates the query heads beside.
 *   rows: rows that the arguments hold, the batch's tokens at least (a replay leaves out tokens behind them);
 *   k, v: element (token, kv head, d) at token x *_tok + head x *_head + d (device; 16-byte aligned, strides multiples
 *         of 8 elements, so k and v may be parts of one projection's rows; any where there is one row, one head);
 *   q:    the same for the q_heads query heads, or NULL; q_out: [tokens][q_heads][head_dim] (device; it may be q, with
 *         those strides, and overlap the arguments in no other way).
 * rotate != 0: K and q are rotated at their tokens' positions by the handle's rope (refused if it has none); 0: K is
 * stored as it is (rows that are rotated already) and q must be NULL. */
int mpg_append(mpg_t* h, int layer, int rows, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
               int64_t v_head, const void* q, int64_t q_tok, int64_t q_head, void* q_out, int rotate);
/* Attention of the batch's tokens over their sequences' pages, one layer. A token at position p sees positions
 * (p - window, p] (window of the layer; 0: [0, p]).
 *   rows:  as mpg_append's;
 *   q:     as mpg_append's; scale > 0: scores are scale q.k;
 *   sinks: NULL, or f32 [q_heads] (device): a logit that joins the softmax's sum but no value;
 *   gate:  NULL, or elements as q's with its own strides: out = attention x sigmoid(gate);
 *   out:   [tokens][q_heads][head_dim] (device), 16-byte aligned; it overlaps no argument.
 * Sums and softmax in f32; the weights are rounded to the cache's type for the matrix units. What stands in positions a
 * token does not see, NaN and infinities included, has no effect on it. */
int mpg_attend(mpg_t* h, int layer, int rows, const void* q, int64_t q_tok, int64_t q_head, float scale, const float* sinks,
               const void* gate, int64_t g_tok, int64_t g_head, void* out);
/* Positions [p0, p1) of a sequence's K or V: dst [p1 - p0][kv_heads][head_dim] of the cache's type (device). When captured,
 * a replay reads the pages the sequence has then as far as the device knows: as of the last mpg_begin or mpg_read_rows. */
int mpg_read_rows(mpg_t* h, int layer, int which, int seq, int p0, int p1, void* dst);

#ifdef __cplusplus
}
#endif
#endif
