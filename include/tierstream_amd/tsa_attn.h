/*
 * tierstream MI355X attention operators: the other half of a layer whose experts this library streams.
 *
 *  - tsa_rotate: queries and keys turned by their positions, and the gradient.
 *  - tsa_cache_plan / tsa_cache_slots: pages, positions and slots of a step's tokens, from the requests' lengths, on the device.
 *  - tsa_cache_store / tsa_cache_load: keys and values to their slots as 4-bit values, and back.
 *  - tsa_attend_cached: the attention of new tokens over the pages of their requests.
 *  - tsa_attend / tsa_attend_backward: attention over packed sequences of 16-bit keys and values, and its gradients.
 *
 * A decode step is rotate, plan (once for all layers), store and attend_cached; with the cache at 4 bits its HBM goes to the
 * experts' slots instead. A prompt is rotate, attend and store; training is rotate, attend and their gradients.
 *
 * As in tsa_ops.h: pointers are device memory, except the argument structs, which are read before the call returns; every launch
 * is asynchronous on `stream` (a hipStream_t, NULL = the null stream), allocates nothing, may be captured into a hipGraph, and
 * gives the same bits for the same inputs. Outputs may not overlap inputs, except where a comment allows it. Return: SS_OK,
 * SS_E_INVALID (argument checks, done on the host before any launch), SS_E_BACKEND (a HIP error).
 *
 * What the device alone can see is checked there and reads or writes nothing out of range: a position below 0, a slot or page out of
 * range and a length below 0 count as none, lengths and sequences end at the arrays they index.
 *
 * Alignment: every array at its element's size, pages and workspaces at 16 bytes. Heads that start 16-byte aligned (base and strides)
 * with a head_dim that is a multiple of 8 are the fastest. Infinities and NaN reach the rows that attend to them and no others; a row may
 * be NaN as a whole, its lse too, for one in a tile of 64 keys that the mask cuts for any of 128 rows, or at a new token of its request (the
 * cache), and so may a key's gradients. Arrays and stream belong to the current device. A workspace belongs to one stream, or to
 * graphs that do not run at once; nothing in it is kept from call to call.
 *
 * Sizes: tokens and sequences below 2^24, pages and a table's width below 2^25, heads up to 1024; tsa_cache_store and _load: tokens x
 * kv_heads x head_dim below 2^33; tsa_attend_cached: tokens x heads below 2^26, and (requests with tokens + tokens x heads / kv_heads /
 * 16) x width below 2^31; tsa_attend and its gradients: tokens x heads below 2^30, sequences x heads below 2^23.
 */
#ifndef TIERSTREAM_AMD_TSA_ATTN_H
#define TIERSTREAM_AMD_TSA_ATTN_H

#include "tsa_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TSA_ROTARY_MAX_PAIRS 128u
#define TSA_CACHE_PAGE 64u           /* tokens of a page */
#define TSA_CACHE_MAX_REQUESTS 4096u
#define TSA_ATTEND_MAX_HEAD_DIM 128u

/* Rows of heads: value i of head h of token t is element t x token_stride + h x head_stride + i. */
typedef struct tsa_heads {
  void* p;
  uint64_t token_stride, head_stride;
  uint32_t heads, reserved;
} tsa_heads;

/* ---- rotary positions ---- */

/* How positions turn a head: pair i of its first `rotated` values by position x f_i radians, f_i = base^(-2 i / rotated).
 * interleaved 0: pair i is values i and i + rotated / 2; 1: values 2 i and 2 i + 1. Behind them values stay as they are.
 * Scaled for contexts `factor` (1: not) times as long as the `trained` ones: with t_i = trained f_i / (2 pi), the turns inside the
 * trained length, f_i is kept where t_i >= high, divided by factor where t_i <= low, and blended by (t_i - low) / (high - low)
 * between (trained 0: all divided). Sines and cosines are multiplied by `amplitude`. */
typedef struct tsa_rotary_params {
  double base, factor, trained, low, high, amplitude;
  uint32_t rotated;        /* even, 2..256 */
  uint32_t interleaved;
} tsa_rotary_params;
/* The same as the kernels take it; made once on the host by tsa_rotary_init. */
typedef struct tsa_rotary {
  double turns[TSA_ROTARY_MAX_PAIRS]; /* f_i / (2 pi) */
  double amplitude;
  uint32_t pairs, interleaved;
} tsa_rotary;
SS_API ss_status tsa_rotary_init(const tsa_rotary_params* p, tsa_rotary* out);

/* y = x turned by its token's position; for one or two arrays (queries and keys; x[1].heads may be 0). backward 1: the gradient,
 * x that of y and y that of x (turned back, and multiplied by the same amplitude). y may be x itself (not a shifted part of it).
 * Rows of tokens whose position is below 0 are not written. Angles are in 64 bits, products in 32. */
typedef struct tsa_rotate_args {
  tsa_heads x[2], y[2];
  const int32_t* positions; /* [tokens] */
  uint32_t tokens, head_dim;
  uint32_t type;            /* TSA_BF16, TSA_F16, TSA_F32 */
  uint32_t backward;
} tsa_rotate_args;
SS_API ss_status tsa_rotate(const tsa_rotary* r, const tsa_rotate_args* a, void* stream);

/* ---- a paged cache of 4-bit keys and values ---- */

/* Pages of 64 tokens, kv_heads of them together; slot s is token s mod 64 of page s / 64. A page of one head, 72 head_dim bytes:
 *   keys [64 tokens][4 g][blocks][4 bytes], key scales [64][blocks], value scales [64][blocks] (half precision), values
 *   [blocks][64 tokens][16 bytes]; blocks = head_dim / 32.
 * A block is 32 values of one token as TSA_Q4 has them: byte j holds value j + 8 in its low half and value 16 + j + 8 in its high
 * half (a key's byte 4 g + i at [g][b][i]), each -8..7 times the block's scale. */
typedef struct tsa_cache {
  void* pages;             /* [n_pages][kv_heads][72 head_dim] bytes */
  uint32_t n_pages;        /* below 2^25 */
  uint32_t kv_heads, head_dim; /* head_dim 32, 64, 96 or 128 */
  uint32_t reserved;
} tsa_cache;

/* The pages, positions and slots of a step. Request i holds lengths[i] tokens on the pages of its table row (entries behind them
 * are not looked at) and gets fresh[i] more, or has ended (fresh[i] < 0: its pages become free, its length 0; the table keeps
 * them until they are overwritten). Free pages are a stack free[0..n_free): ended requests push theirs in order, then requests in order
 * take the pages they lack from its end. ends[i] is the new length, left the pages left on the stack, first[i] the tokens before
 * request i's in this step (first[requests]: all of them); token r of request i has position lengths[i] + r and row first[i] + r
 * of positions and slots. Rows behind the last get -1 in both.
 * All or nothing: where status is not 0 (1: pages short, 2: rows short, 4: a table row too short, 8: a length below 0 or a stack
 * out of its bounds; the sum of those that apply) table, stack and lengths stay, and no request gets a token.
 * ends may be lengths and left may be n_free. */
typedef struct tsa_cache_plan_args {
  const int32_t* lengths;  /* [requests] */
  const int32_t* fresh;    /* [requests] */
  int32_t* table;          /* [requests][width] page numbers */
  uint64_t table_stride;
  int32_t* free;           /* [pages] */
  const int32_t* n_free;   /* [1] */
  int32_t* ends;           /* [requests] */
  int32_t* left;           /* [1] */
  int32_t* first;          /* [requests + 1] */
  int32_t* positions;      /* [rows] */
  int32_t* slots;          /* [rows] */
  int32_t* status;         /* [1] */
  uint32_t requests, width, pages, rows;
} tsa_cache_plan_args;
SS_API ss_status tsa_cache_plan(const tsa_cache_plan_args* a, void* stream);

/* The same positions and slots for requests whose pages are there: the rows first[i]..first[i + 1] are the tokens of request i that
 * end with its length ends[i] (its whole context where first counts whole lengths). Reads table, ends, first, requests, width and
 * rows of the struct, writes positions and slots. A row that has no page (-1 in the table, before the first token) gets slot -1, one before
 * first[0] or behind the last one -1 in both. */
SS_API ss_status tsa_cache_slots(const tsa_cache_plan_args* a, void* stream);

/* Token t's keys and values to slot slots[t]. A block's scale is its value of the largest size (of equal ones the first) over -8,
 * rounded to half precision; values are rounded to the nearest whole step of it, ties to even. Blocks with an infinity, a NaN or a
 * scale beyond half precision read as NaN. Slots out of range are skipped; one that is given twice holds a mixture. */
typedef struct tsa_cache_rows_args {
  tsa_heads k, v;          /* kv_heads heads of head_dim values */
  const int32_t* slots;    /* [tokens] */
  uint32_t tokens;
  uint32_t type;           /* TSA_BF16 or TSA_F16 */
} tsa_cache_rows_args;
SS_API ss_status tsa_cache_store(const tsa_cache* c, const tsa_cache_rows_args* a, void* stream);
/* Back from their slots, rounded to type. Rows of slots out of range are not written. */
SS_API ss_status tsa_cache_load(const tsa_cache* c, const tsa_cache_rows_args* a, void* stream);

/* out_t = sum_j p_tj v_j, p_t the softmax of scale q_t . k_j over the keys j that token t attends to. Request i's tokens are
 * the rows first[i]..first[i + 1]; they are the last ones of its length ends[i] (stored before the call), and each attends to
 * the tokens up to itself. Query head h reads kept head h / (heads / kv_heads). A row without keys is 0; rows behind the last request
 * are left as they were. A token on a page out of range counts as absent. For one or a few tokens a request; it
 * holds for any number. Probabilities times their values' scales are rounded to half precision, in ranges of their own (a scale below 2^-15
 * of the largest of its block of the request keeps fewer bits; with TSA_BF16 probabilities are before that, too); all sums are in 32 bits. */
typedef struct tsa_attend_cached_args {
  tsa_heads q, out;        /* heads a multiple of kv_heads */
  const int32_t* table;    /* [requests][width] */
  uint64_t table_stride;
  const int32_t* ends;     /* [requests] */
  const int32_t* first;    /* [requests + 1] */
  uint32_t tokens, requests, width;
  uint32_t type;           /* TSA_BF16 or TSA_F16 */
  float scale;
  uint32_t reserved;
} tsa_attend_cached_args;
/* Grows with tokens, requests and width. */
SS_API uint64_t tsa_attend_cached_workspace(const tsa_cache* c, const tsa_attend_cached_args* a);
SS_API ss_status tsa_attend_cached(const tsa_cache* c, const tsa_attend_cached_args* a, void* workspace, uint64_t workspace_bytes,
                                   void* stream);

/* ---- attention over packed sequences ---- */

/* out_t = sum_j p_tj v_j, p_t the softmax of scale q_t . k_j over the keys of t's sequence: with n queries and m keys, all of them,
 * or (causal) those up to j = i + m - n for the sequence's query i. A row without keys is 0 (its lse -infinity); rows behind the
 * last sequence are left as they were. Query head h reads key head h / (heads / kv_heads). Probabilities are rounded to type (in half
 * precision times 2^15), and in sequences of at most 2^17 pairs of a query and a key what that leaves of them is multiplied too; all sums
 * are in 32 bits. */
typedef struct tsa_attend_args {
  tsa_heads q, k, v, out;
  const int32_t* first;    /* [sequences + 1]: a sequence's first query row; ascending from 0. NULL: one sequence of all rows */
  const int32_t* k_first;  /* the same of its keys; NULL: first */
  float* lse;              /* [heads][tokens]: log sum exp of each row's scaled scores, or NULL (the backward pass reads it) */
  uint32_t tokens, k_tokens, sequences;
  uint32_t head_dim;       /* a multiple of 8, 8..128 */
  uint32_t type;           /* TSA_BF16 or TSA_F16 */
  uint32_t causal;
  float scale;
  uint32_t reserved;
} tsa_attend_args;
SS_API ss_status tsa_attend(const tsa_attend_args* a, void* stream);

/* The gradients for dout, from the forward call's inputs, out and lse. dq, or dk and dv together, may be absent (p NULL). Keys that
 * no query attends to get 0; rows behind the last sequence are left as they were. Probabilities and the scores' gradients are rounded
 * as tsa_attend's probabilities are (the latter in half precision behind a power of two that the largest of a row so far chooses); all sums
 * are in 32 bits. A row's sum_j p_j dout . v_j is added up where its tile of 128 queries attends to at most 512 keys, and taken as dout . out
 * beyond. */
typedef struct tsa_attend_grad_args {
  tsa_attend_args f;
  tsa_heads dout, dq, dk, dv;
} tsa_attend_grad_args;
SS_API uint64_t tsa_attend_backward_workspace(const tsa_attend_args* f);
SS_API ss_status tsa_attend_backward(const tsa_attend_grad_args* a, void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TIERSTREAM_AMD_TSA_ATTN_H */
