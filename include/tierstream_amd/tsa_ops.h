/*
 * tierstream MI355X operators: what an engine computes with the weight units this library puts in HBM.
 *
 *  - tsa_route / tsa_route_backward: the experts of each row from the router's logits. The ids are what
 *    ss_dg_enqueue_export and ss_layer_routes take, ids and weights what tsa_ffn takes.
 *  - tsa_linear: a product with streamed (or any) weights, with bias, activation and residual in its epilogue.
 *  - tsa_ffn / tsa_ffn_backward: the gated feed-forward blocks of the chosen experts, their weights read where they
 *    are: the slots of a device-gated arena (through ss_dg_slot), the addresses of the host contract's table, or
 *    stacked arrays.
 *
 * Matrices are row-major with contiguous rows; a stride counts elements from row to row. Pointers are device memory,
 * except the argument structs, which are read before the call returns. Every launch is asynchronous on `stream` (a
 * hipStream_t, NULL = the null stream), allocates nothing, may be captured into a hipGraph, and gives the same bits
 * for the same inputs. Outputs may not overlap inputs, except where a residual is the output itself. Return: SS_OK,
 * SS_E_INVALID (argument checks, done on the host before any launch), SS_E_BACKEND (a HIP error).
 *
 * Alignment: every matrix at its element's size, workspaces at 16 bytes, the units of a table at 16 (their addresses are the
 * device's, no call can look at them; a descriptor's unit_align is 256 unless it says otherwise, and has to be 16 at least). Rows
 * that start 16-byte aligned (base and stride) and hold a multiple of 8 values are the fastest. 4-bit weights outside a table: 4
 * bytes; 16 is faster.
 *
 * Infinities and NaN stay in the rows they stand in, and what an id, a table entry or a logit masks is not read. With 4-bit
 * weights (whose scales are finite) an infinity in a row of x may give NaN where the formula gives an infinity.
 */
#ifndef TIERSTREAM_AMD_TSA_OPS_H
#define TIERSTREAM_AMD_TSA_OPS_H

#include "../strix_stream/ss.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. TSA_Q4 (weights only, the descriptor's part format Q4_0): rows of 18-byte blocks of 32 values, a
 * half-precision scale s, then 16 bytes; value i is (low half of byte i - 8) x s, value 16 + i the high half's. */
enum { TSA_BF16 = 0, TSA_F16 = 1, TSA_F32 = 2, TSA_Q4 = 3 };
/* Activations: identity (tsa_linear only), v / (1 + exp(-v)), v Phi(v), its tanh form, max(v, 0). */
enum { TSA_ACT_NONE = 0, TSA_ACT_SILU = 1, TSA_ACT_GELU = 2, TSA_ACT_GELU_TANH = 3, TSA_ACT_RELU = 4 };

#define TSA_ROUTE_MAX_EXPERTS 1024u
#define TSA_ROUTE_MAX_TOP_K 64u
#define TSA_FFN_MAX_EXPERTS 512u

/* The top_k largest logits of each row, largest first, ties to the lower id. With m the row's largest logit and
 * e_i = exp(logit_i - m): weights_j = scale x e_{ids_j} / sum, the sum over the chosen ones (renorm = 1) or over all
 * (renorm = 0). A logit of -infinity or NaN is a masked expert: never chosen, and 0 in the sums. Where fewer than
 * top_k are left (a row may be masked whole), the rest are id -1 with weight 0. */
typedef struct tsa_route_args {
  const void* logits;      /* [rows][n_experts] */
  uint64_t logits_stride;
  int32_t* ids;            /* [rows][top_k] */
  float* weights;          /* [rows][top_k] */
  uint32_t rows, n_experts, top_k;
  uint32_t type;           /* of the logits: TSA_F32, TSA_BF16, TSA_F16 */
  uint32_t renorm;
  float scale;
} tsa_route_args;
SS_API ss_status tsa_route(const tsa_route_args* a, void* stream);

/* dlogits from the gradient of the weights, for the ids that tsa_route gave (ids of -1 take no gradient; masked
 * experts get 0). `weights` of the struct is not read. */
SS_API ss_status tsa_route_backward(const tsa_route_args* a, const float* dweights, void* dlogits,
                                    uint64_t dlogits_stride, void* stream);

/* y = act(x W^T + bias) + residual. */
typedef struct tsa_linear_args {
  const void* x;           /* [rows][n_in] of x_type */
  uint64_t x_stride;
  const void* w;           /* [n_out][n_in] of w_type; TSA_Q4: whole blocks, rows back to back */
  uint64_t w_stride;       /* (TSA_Q4: n_in) */
  const void* bias;        /* [n_out] of x_type, or NULL */
  const void* residual;    /* [rows][n_out] of y_type, or NULL; may be y */
  uint64_t residual_stride;
  void* y;                 /* [rows][n_out] of y_type */
  uint64_t y_stride;
  uint32_t rows, n_in, n_out;
  uint32_t x_type;         /* TSA_BF16 or TSA_F16 */
  uint32_t w_type;         /* x_type or TSA_Q4 (n_in a multiple of 32) */
  uint32_t y_type;         /* x_type or TSA_F32 */
  uint32_t act;
  uint32_t reserved;
} tsa_linear_args;
/* Workspace bytes of a call (0: none is used): where more than a few rows are to be multiplied and rows of x or w do not
 * start 16-byte aligned or are no multiple of 8 values, these are packed first. Sizes are below 2^24, rows x n_out below 2^37. */
SS_API uint64_t tsa_linear_workspace(const tsa_linear_args* a);
SS_API ss_status tsa_linear(const tsa_linear_args* a, void* workspace, uint64_t workspace_bytes, void* stream);

/* The weights of a layer's experts: part 0 (gate) and 1 (up) are [d_ff][d_model], part 2 (down) is [d_model][d_ff].
 * Exactly one of part[0], table and view says where they are. */
typedef struct tsa_experts {
  uint32_t n_experts, d_model, d_ff;
  uint32_t w_type;                 /* TSA_BF16, TSA_F16, TSA_Q4 (d_model and d_ff multiples of 32) */
  const void* part[3];             /* expert e's part p at part[p] + e x part_stride[p] bytes */
  uint64_t part_stride[3];
  const uint64_t* table;           /* ss_layer_view.table_dev: expert e's unit (its parts back to back) at table[e];
                                      an entry of 0 (not acquired) counts as no expert, every other is 16-byte aligned */
  const ss_dg_device_view* view;   /* host struct, copied: gated layer `gated`, read behind its ss_dg_enqueue_wait */
  uint32_t gated, reserved;
} tsa_experts;

/* y_t = residual_t + sum_j weights_tj x down (act(gate x_t) * (up x_t)), the weights of expert ids_tj. An id below 0 or
 * from n_experts up adds nothing; a row may have none. ids NULL: every row through expert 0 (top_k 1).
 * All sums are in 32 bits; act(gate x) * (up x) is rounded once to 16 (with its weight, where there is one row), in half
 * precision behind a power of two that its row's largest value chooses, so that nothing that 32 bits hold overflows or is lost. */
typedef struct tsa_ffn_args {
  const void* x;           /* [rows][d_model] of type */
  uint64_t x_stride;
  const int32_t* ids;      /* [rows][top_k], or NULL */
  const float* weights;    /* [rows][top_k], or NULL: 1 */
  const void* residual;    /* [rows][d_model] of type, or NULL; may be y */
  uint64_t residual_stride;
  void* y;                 /* [rows][d_model] of type */
  uint64_t y_stride;
  uint32_t rows, top_k;
  uint32_t type;           /* TSA_BF16 or TSA_F16; the experts' w_type is the same or TSA_Q4 */
  uint32_t act;            /* not TSA_ACT_NONE */
} tsa_ffn_args;
SS_API uint64_t tsa_ffn_workspace(const tsa_experts* e, uint32_t rows, uint32_t top_k);
SS_API ss_status tsa_ffn(const tsa_experts* e, const tsa_ffn_args* a, void* workspace, uint64_t workspace_bytes,
                         void* stream);

/* The gradients of tsa_ffn for dy (the residual's gradient is dy itself). Nothing of the forward pass is kept: gate x and
 * up x are computed again, in 32 bits. The experts' w_type is args' type (4-bit weights have no backward pass).
 * All sums are in 32 bits; of what lies between them the gradients of gate x and up x, and the weighted act(gate x) * (up x), are
 * rounded once to 16 bits, in half precision behind a power of two that the largest value of the expert's rows chooses. */
typedef struct tsa_ffn_grad_args {
  const void* x;           /* [rows][d_model] of type */
  uint64_t x_stride;
  const int32_t* ids;      /* as in tsa_ffn_args */
  const float* weights;
  const void* dy;          /* [rows][d_model] of type */
  uint64_t dy_stride;
  void* dx;                /* [rows][d_model] of type, or NULL */
  uint64_t dx_stride;
  float* dweights;         /* [rows][top_k], or NULL; 0 where an id adds nothing */
  void* dgate;             /* [n_experts][d_ff][d_model] of type, back to back; the three together, or all NULL */
  void* dup;
  void* ddown;             /* [n_experts][d_model][d_ff] */
  uint32_t rows, top_k;
  uint32_t type, act;
} tsa_ffn_grad_args;
SS_API uint64_t tsa_ffn_backward_workspace(const tsa_experts* e, uint32_t rows, uint32_t top_k);
SS_API ss_status tsa_ffn_backward(const tsa_experts* e, const tsa_ffn_grad_args* a, void* workspace,
                                  uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TIERSTREAM_AMD_TSA_OPS_H */
