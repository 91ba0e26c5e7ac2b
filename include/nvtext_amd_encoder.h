/*
 * nvtext_amd_encoder.h -- C ABI of the operators between wordpiece_tokenize's column of ids and a model that learns
 * from it: embedding of a LIST<INT32> column, dropout, layer norm, the matrix product of a layer (linear), rotary positions
 * and attention, each with its gradient.  The tokens of all rows lie one after the other (packed); every operator but the
 * embedding, rotary positions and attention treats a token by itself.
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

/* The heads of packed tokens: value j of head h of token t lies at data[t * stride + h * head_stride + j], so that those of
 * queries, keys and values can be parts of the rows of one matrix.  stride and head_stride are in values and not negative;
 * each is of no meaning where there are fewer than two tokens or heads.  data is aligned to its element type.  Heads of a width that is a multiple of
 * 8, with both strides multiples of 8 and data at a multiple of 16 bytes, are read fastest (FLOAT32: of 4 each). */
typedef struct nvtext_amd_heads {
  void* data; /* device; may be NULL when there are no values */
  int64_t tokens;
  int64_t heads;
  int64_t width;
  int64_t stride;
  int64_t head_stride;
  int32_t type; /* NVTEXT_AMD_TYPE_FLOAT32, _FLOAT16 or _BFLOAT16 */
} nvtext_amd_heads;

typedef enum nvtext_amd_rotary_layout {
  NVTEXT_AMD_ROTARY_HALF        = 0, /* pair n of N is values n and n + N of a head */
  NVTEXT_AMD_ROTARY_INTERLEAVED = 1  /* pair n is values 2 n and 2 n + 1 */
} nvtext_amd_rotary_layout;

/* Rotary positions: of every head of a token at position t of its row, pair n of the first 2 * pairs values (a, b) becomes
 *   magnitude * (a cos w - b sin w, a sin w + b cos w),  w = t * frequencies[n], and with `inverse` w = -t * frequencies[n];
 * the values behind them are copied.  The inverse call with the same magnitude, on the gradient of out, is the backward pass.
 * Row r's tokens are offsets[r] up to offsets[r + 1] (device, rows + 1 values, ascending); their positions count from
 * starts[r] on (device, `rows` values; NULL: from 0 on).  A token that belongs to no row is copied.  frequencies: `pairs` values on
 * the device, radians a position.  Angles are computed in 64 bits and reduced to a part of a turn before they lose any, so positions may be
 * as far as they come: sine and cosine are off by 2^-22 at most (at position t by t * |frequency| * 2^-51 more); products and sums are
 * held in 32 bits and rounded once.  out has x's shape and type, and may be x, but not hold values of it in other places. */
nvtext_amd_status nvtext_amd_rotary(const nvtext_amd_heads* x,
                                    int32_t rows,
                                    const int32_t* offsets,
                                    const int32_t* starts,
                                    const double* frequencies,
                                    int64_t pairs,
                                    int32_t layout,
                                    int32_t inverse,
                                    double magnitude,
                                    void* stream,
                                    const nvtext_amd_heads* out);

/* Attention: every head of a token looks at the keys of its row.
 * Row r has the tokens offsets[r] up to offsets[r + 1] of q, and of k and v those from key_offsets[r] on, key_lengths[r] of
 * them, or up to key_offsets[r + 1] where key_lengths is NULL (all on the device; offsets ascend, rows + 1 values each; key_offsets
 * NULL: k and v have q's tokens and offsets).  With key_lengths, keys may lie in places with room for more, which is not read.
 * Head h of q sees head h / (q's heads / k's heads) of k and v, whose heads are a divisor of q's.  Token i of Q in a row sees key j of K
 * there, for causal = 0 every one, else j <= i + K - Q: its last token all of them.  Over the keys it sees, with s_j = scale * (q . k_j),
 *   logsum = log(sum of exp(s_j)),  out = sum of exp(s_j - logsum) * v_j;
 * a token that sees none, or belongs to no row, has zeros in out and -infinity in logsum.  What a token does not see is without
 * effect on it, whatever it is, NaN too.  (Of a result that cannot be finite for what its token sees, it is not laid down whether it is an infinity or NaN.  Of
 * causal rows, infinities or NaN that all over the values or the gradient lie among what is finite cost a lot of time.)
 * q, k, v and out are of one type and width, of at most 256 values, in at most 65536 heads of 2^31 - 1025 tokens; scale is not negative.  logsum (NULL: not wanted; the gradient needs it)
 * has a value of FLOAT32 at [h * tokens + t].  rest (NULL: not wanted; FLOAT32 has none), of a value for each of out's, [heads, tokens, width]
 * one after the other: what rounding left off it, in 8 bits, for the gradient.  Products, exponentials' sums and out are held in 32 bits; of 16-bit types, the exponentials are
 * rounded to the type before they are multiplied with v, as the matrix cores take them, and out is divided by their sum as they are then
 * (logsum is that of the values before). */
nvtext_amd_status nvtext_amd_attention(const nvtext_amd_heads* q,
                                       const nvtext_amd_heads* k,
                                       const nvtext_amd_heads* v,
                                       int32_t rows,
                                       const int32_t* offsets,
                                       const int32_t* key_offsets,
                                       const int32_t* key_lengths,
                                       int32_t causal,
                                       double scale,
                                       void* stream,
                                       const nvtext_amd_allocator* mr,
                                       const nvtext_amd_heads* out,
                                       float* logsum,
                                       int8_t* rest);

/* The gradients of attention from grad, that of its out, and from its out, logsum and rest, over the same rows.  (rest may be NULL: the
 * gradients of q and k are off by a rounding of out more, then.)  With p = exp(s - logsum)
 * and d = p * (grad . v - grad . out), for every token and the keys it sees, each rounded to the type before it is multiplied:
 *   q_grad = scale * sum over the keys of d * k,
 *   k_grad = scale * sum over the tokens, and the heads that see one, of d * q,  v_grad = the same sum of p * grad.
 * All three are wanted, whole: keys that nobody sees, or that belong to no row, have zeros.  They may be parts of one matrix' rows, as q, k and v
 * may, but overlap no input. */
nvtext_amd_status nvtext_amd_attention_backward(const nvtext_amd_heads* grad,
                                                const nvtext_amd_heads* q,
                                                const nvtext_amd_heads* k,
                                                const nvtext_amd_heads* v,
                                                const nvtext_amd_heads* out,
                                                const float* logsum,
                                                const int8_t* rest,
                                                int32_t rows,
                                                const int32_t* offsets,
                                                const int32_t* key_offsets,
                                                const int32_t* key_lengths,
                                                int32_t causal,
                                                double scale,
                                                void* stream,
                                                const nvtext_amd_allocator* mr,
                                                const nvtext_amd_heads* q_grad,
                                                const nvtext_amd_heads* k_grad,
                                                const nvtext_amd_heads* v_grad);

#ifdef __cplusplus
}
#endif
#endif /* NVTEXT_AMD_ENCODER_H */
