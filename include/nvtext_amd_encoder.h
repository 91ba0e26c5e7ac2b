/*
 * nvtext_amd_encoder.h -- C ABI of the operators between wordpiece_tokenize's column of ids and a model that learns
 * from it: embedding of a LIST<INT32> column, dropout, layer norm and the matrix product of a layer (linear), each with
 * its gradient.  The tokens of all rows lie one after the other (packed); every operator but the embedding treats a
 * token by itself.
 *
 * The conventions are those of nvtext_amd.h: device pointers, the caller's stream, status codes, the text of the last
 * error.  Matrices are views of the caller's memory, the results too (their sizes are known before the call);
 * temporaries come from the nvtext_amd_allocator.  No call waits for the device, and none reads a result of an earlier
 * call but what is passed to it.  A result may not overlap an input, with the exceptions named below.  Sums are held in
 * 32 bits and added in an order that depends on sizes (the embedding's gradients: on the column too) and the device's
 * number of CUs alone, not on where matrices lie or how far apart their rows are: the same inputs give the same bits.
 */
#ifndef NVTEXT_AMD_ENCODER_H
#define NVTEXT_AMD_ENCODER_H

#include "nvtext_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of a matrix: NVTEXT_AMD_TYPE_FLOAT32 and these two, which cudf::type_id has no values for. */
enum {
  NVTEXT_AMD_TYPE_FLOAT16  = 101,
  NVTEXT_AMD_TYPE_BFLOAT16 = 102
};

/* `rows` rows of `cols` values, one row every `stride` values (stride >= cols; of no meaning for fewer than two rows).
 * data is aligned to its element type; matrices whose rows all begin at multiples of 16 bytes are read fastest.
 * A vector is a matrix of one row. */
typedef struct nvtext_amd_matrix {
  void*   data; /* device; may be NULL when there are no values */
  int64_t rows;
  int64_t cols;
  int64_t stride;
  int32_t type; /* NVTEXT_AMD_TYPE_FLOAT32, _FLOAT16 or _BFLOAT16 */
} nvtext_amd_matrix;

/* out[t] = token_table[id of t] + position_table[place of t in its row], in 32 bits, rounded once.  `tokens` is a result
 * of nvtext_amd_wordpiece_tokenize (or any LIST<INT32> column: size, offsets, child and child_size are read).  A token
 * whose id is no row of the table (the -1 of a vocabulary without "[UNK]" among them) takes nothing from it, a token
 * further from its row's start than position_table has rows takes nothing from that; a value of the child that belongs
 * to no row gives zeros.  position_table: NULL for none.  out has child_size rows; the three matrices are of one type
 * and width. */
nvtext_amd_status nvtext_amd_embedding(const nvtext_amd_list_column* tokens,
                                       const nvtext_amd_matrix* token_table,
                                       const nvtext_amd_matrix* position_table,
                                       void* stream,
                                       const nvtext_amd_matrix* out);

/* The gradients of both tables, whole: rows that no token took from are zeros.  grad has child_size rows.  token_grad
 * and position_grad (NULL: not wanted) are of grad's type or FLOAT32. */
nvtext_amd_status nvtext_amd_embedding_backward(const nvtext_amd_list_column* tokens,
                                                const nvtext_amd_matrix* grad,
                                                void* stream,
                                                const nvtext_amd_allocator* mr,
                                                const nvtext_amd_matrix* token_grad,
                                                const nvtext_amd_matrix* position_grad);

/* out = x * 65536 / (65536 - T) where x is kept and 0 where it is dropped, T = p * 65536 rounded: value (i, j) is
 * dropped where its draw is less than T.  Its draw is the 16-bit half j % 2 (the low one first) of word j % 8 / 2 of
 * Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the
 * counter {j / 8, i mod 2^32, i / 2^32, offset} and the key {seed mod 2^32, seed / 2^32}.  No mask is stored: the same
 * call on the gradient of out is the backward pass.  p = 1 drops everything; a value that is dropped may be anything,
 * NaN too.  out may be x. */
nvtext_amd_status nvtext_amd_dropout(const nvtext_amd_matrix* x,
                                     double p,
                                     uint64_t seed,
                                     uint32_t offset,
                                     void* stream,
                                     const nvtext_amd_matrix* out);

/* s = residual + dropout(x) (residual: NULL for none; p = 0: nothing is dropped), then over each row
 * mean = sum(s) / cols, rstd = 1 / sqrt(sum((s - mean)^2) / cols + eps), out = (s - mean) * rstd * weight + bias.
 * x, residual, out and sum are of one type; weight and bias, of cols values each, of that type or FLOAT32.
 * What the gradient needs is written where it is asked for: sum (s, rounded; the statistics are those of s before it is
 * rounded) and the rows' mean and rstd (FLOAT32, all NULL or as wanted).  out and sum may each be x or the residual. */
nvtext_amd_status nvtext_amd_layer_norm(const nvtext_amd_matrix* x,
                                        const nvtext_amd_matrix* residual,
                                        const nvtext_amd_matrix* weight,
                                        const nvtext_amd_matrix* bias,
                                        double eps,
                                        double p,
                                        uint64_t seed,
                                        uint32_t offset,
                                        void* stream,
                                        const nvtext_amd_matrix* out,
                                        const nvtext_amd_matrix* sum,
                                        float* mean,
                                        float* rstd);

/* The gradients of layer_norm.  grad is that of out, sum_grad (NULL for none) that of s where s goes on to the next
 * block.  With h = (sum - mean) * rstd and a = grad * weight:
 *   residual_grad = rstd * (a - sum(a) / cols - h * sum(a * h) / cols) + sum_grad
 *   x_grad        = dropout(residual_grad), which with p = 0 is residual_grad: x_grad may be NULL then
 *   weight_grad   = the sum over the rows of grad * h, bias_grad that of grad (both NULL or both wanted; of weight's type).
 * residual_grad may be grad, sum or sum_grad. */
nvtext_amd_status nvtext_amd_layer_norm_backward(const nvtext_amd_matrix* grad,
                                                 const nvtext_amd_matrix* sum,
                                                 const float* mean,
                                                 const float* rstd,
                                                 const nvtext_amd_matrix* weight,
                                                 const nvtext_amd_matrix* sum_grad,
                                                 double p,
                                                 uint64_t seed,
                                                 uint32_t offset,
                                                 void* stream,
                                                 const nvtext_amd_allocator* mr,
                                                 const nvtext_amd_matrix* x_grad,
                                                 const nvtext_amd_matrix* residual_grad,
                                                 const nvtext_amd_matrix* weight_grad,
                                                 const nvtext_amd_matrix* bias_grad);

typedef enum nvtext_amd_activation {
  NVTEXT_AMD_ACTIVATION_NONE      = 0,
  NVTEXT_AMD_ACTIVATION_RELU      = 1, /* max(z, 0) */
  NVTEXT_AMD_ACTIVATION_GELU      = 2, /* z * (1 + erf(z / sqrt 2)) / 2 */
  NVTEXT_AMD_ACTIVATION_GELU_TANH = 3, /* z * (1 + tanh(sqrt(2 / pi) * (z + 0.044715 z^3))) / 2 */
  NVTEXT_AMD_ACTIVATION_SILU      = 4  /* z / (1 + exp(-z)) */
} nvtext_amd_activation;

/* z = x * weight^T + bias, out = activation(z) + residual, in 32 bits, each rounded once.  x: rows of `inputs` values,
 * weight: [outputs, inputs], bias: `outputs` values or NULL, residual: like out or NULL, preactivation: where z is
 * wanted (for the gradient), else NULL.  All of one type.  out may be the residual. */
nvtext_amd_status nvtext_amd_linear(const nvtext_amd_matrix* x,
                                    const nvtext_amd_matrix* weight,
                                    const nvtext_amd_matrix* bias,
                                    int32_t activation,
                                    const nvtext_amd_matrix* residual,
                                    void* stream,
                                    const nvtext_amd_allocator* mr,
                                    const nvtext_amd_matrix* out,
                                    const nvtext_amd_matrix* preactivation);

/* The gradients of linear (that of the residual is grad itself): with d = grad * activation'(preactivation), rounded to
 * the type of the matrices before it is multiplied (of 16-bit types and with an activation x_grad and weight_grad are off by two
 * roundings of that type, then, instead of one),
 *   x_grad = d * weight, weight_grad = d^T * x, bias_grad = the sum over the rows of d (before it is rounded);
 * each NULL where it is not wanted.  preactivation may be NULL for NVTEXT_AMD_ACTIVATION_NONE, where d is grad. */
nvtext_amd_status nvtext_amd_linear_backward(const nvtext_amd_matrix* grad,
                                             const nvtext_amd_matrix* x,
                                             const nvtext_amd_matrix* weight,
                                             int32_t activation,
                                             const nvtext_amd_matrix* preactivation,
                                             void* stream,
                                             const nvtext_amd_allocator* mr,
                                             const nvtext_amd_matrix* x_grad,
                                             const nvtext_amd_matrix* weight_grad,
                                             const nvtext_amd_matrix* bias_grad);

#ifdef __cplusplus
}
#endif
#endif /* NVTEXT_AMD_ENCODER_H */
