/* fhe_ssm_clear.h -- what the client of the encrypted step computes in the clear (libfhe_ssm_clear.so).
 *
 * An encrypted step answers with one hidden row per conversation lane.  The client turns the rows into logits (the
 * vocabulary head stays on its side) and draws the next tokens; between encrypted steps it may draft tokens with a small
 * recurrent model of its own, whose constant-size state is of the same kind as the encrypted one (the reference keeps its
 * plain recurrent companions in spec_decode/).  The operators of those programs are here, as HIP kernels for gfx950:
 *
 *   linear attention   the recurrence of the draft model, with a decay for each head: over a prompt, and over one token
 *   4-bit products     rows times a matrix of 4-bit codes with group scales: the head, and the draft's projections
 *   sampling           the draw of a token under temperature, top-k, top-p and min-p, from given random numbers
 *
 * The draft is worth as much as it foresees what the encrypted model answers, so the client scores answered tokens with it
 * and trains it on them (the reference trains its models in ml-eval/train_fhe_native_ssm.py).  For that, each with its gradient:
 *
 *   layer norm         over the channels of rows
 *   gated recurrence   h <- sigmoid(z) h + sigmoid(-z) x per channel: over a prompt, backwards, and over one token
 *   embedding          rows of a table by token
 *   log-probabilities  of given tokens, with entropy and the most likely alternatives
 *   AdamW              the step over all tensors of a model, with states in 32 or 8 bits
 *
 * Device pointers may come from any HIP allocator and belong to the current device.  Every call that computes takes a
 * hipStream_t (as void*, NULL is the null stream), issues its work there and returns without waiting; no call allocates
 * or copies to the host, and calls may be recorded into a graph.  Sums, states and statistics are held in 32 bits or
 * more.  Results do not depend on how work was scheduled: there is no floating-point atomic.
 * Status codes are ckks_engine.h's; fhe_ssm_clear_last_error() explains the last failure on this thread.  Sizes that a
 * host can see are checked; what lies in device memory (lengths, sampling parameters) is bounded by the kernels.
 */
#ifndef FHE_SSM_CLEAR_H
#define FHE_SSM_CLEAR_H

#include <stddef.h>
#include <stdint.h>

#include "ckks_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of rows, logits, queries, keys, values and scales */
#define FHE_SSM_F32 0
#define FHE_SSM_BF16 1
#define FHE_SSM_F16 2

const char* fhe_ssm_clear_last_error(void);

/* ---- linear attention with a decay for each head ------------------------------------------------------------------
 * Per lane and head, with the state S in R^{dk x dv} (float32) and the log decay g_t <= 0:
 *     S_t = exp(g_t) S_{t-1} + k_t v_t^T        o_t = scale * q_t S_t
 * lanes and tokens may be 0.  dk <= 128, tokens <= 2^24, lanes * heads * ceil(dv / 32) < 2^24.  Shared heads: head h reads
 * query head h / (heads / q_heads) and key head h / (heads / k_heads); values, decays, outputs and states are per head.
 * Strides are in elements, in the order lane, token, head, and may be any (0 shares one row among many), except that
 * different output rows must not overlap; channels are contiguous.  State: [lanes][heads][dk][dv], contiguous;
 * state_in null means zero, state_out null drops the new state, and the two may be the same buffer.  out must overlap
 * no input.  A decay of -inf clears a finite state; one below -1000 is taken as that.  What is not finite in an input
 * reaches its own lane's heads from its token on, and nothing before; there an infinity may come out as NaN. */
typedef struct {
    uint32_t type; /* of q, k, v and out */
    uint32_t lanes, tokens, heads, q_heads, k_heads, dk, dv;
    float scale;
    int64_t q_stride[3], k_stride[3], v_stride[3], decay_stride[3], out_stride[3];
} fhe_ssm_linear_attention;

/* Device memory that a prompt of these sizes needs (0 for many: then workspace may be null). */
int fhe_ssm_linear_attention_workspace(const fhe_ssm_linear_attention* a, size_t* bytes);

/* A prompt.  lengths (int32[lanes] on the device, or null): lane b has lengths[b] tokens (held to [0, tokens]); the rows
 * past them are not read, give zero outputs and leave the state alone. */
int fhe_ssm_linear_attention_prompt(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                    const float* log_decay, const int32_t* lengths, const float* state_in,
                                    float* state_out, void* out, void* workspace, size_t workspace_bytes,
                                    void* stream);

/* One token for every lane: the same with tokens = 1 and no lengths. */
int fhe_ssm_linear_attention_step(const fhe_ssm_linear_attention* a, const void* q, const void* k, const void* v,
                                  const float* log_decay, const float* state_in, float* state_out, void* out,
                                  void* stream);

/* ---- products with 4-bit weights and group scales -----------------------------------------------------------------
 *     y[r][o] = sum_j scale[o][j / group] (code[o][j] - zero[o][j / group]) x[r][j]
 * Codes 0..15, two in a byte (the lower index in the low four bits), rows of (in + 1) / 2 bytes; zero points 0..15 per
 * group, or 8 throughout; the last group may be cut short.  group is 32, 64 or a multiple of 128, rows <= 2^20,
 * ceil(out / 16) * ceil(in / 128) < 2^24.
 * The matrix is laid out once (fhe_ssm_q4_arrange) in the order the kernel reads it; bf16 scales are widened to float32
 * there, float16 ones stay.  Codes and zero points are used exactly; float32 rows are used to their full 24 bits.
 * Sums go through codes held as 16 + c: a row of x with an infinity or a NaN gives NaN in all its outputs and leaves other
 * rows alone, and a row's magnitudes have to sum to less than 2^122 in every group, or its outputs may be NaN. */
typedef struct {
    uint32_t out, in, group;
    uint32_t scale_type; /* of the scales given to fhe_ssm_q4_arrange */
    uint32_t has_zeros;
} fhe_ssm_q4_matrix;

int fhe_ssm_q4_bytes(const fhe_ssm_q4_matrix* m, size_t* bytes); /* of the arranged weights */

/* code_stride: bytes from one row of codes to the next; scales and zeros are [out][ceil(in / group)], contiguous, zeros
 * null unless has_zeros; zero points above 15 are cut to their low four bits. */
int fhe_ssm_q4_arrange(const fhe_ssm_q4_matrix* m, const uint8_t* codes, int64_t code_stride, const void* scales,
                       const uint8_t* zeros, void* weights, void* stream);

/* x: rows of `in` elements, y: rows of `out` elements, both of `type`, strides in elements from row to row. */
int fhe_ssm_q4_product(const fhe_ssm_q4_matrix* m, const void* weights, uint32_t type, uint32_t rows, const void* x,
                       int64_t x_stride, void* y, int64_t y_stride, void* stream);

/* ---- sampling -----------------------------------------------------------------------------------------------------
 * Per row, in the order of falling logits (equal ones by rising index): top-k keeps the first k; with
 * p = softmax(logits / temperature) over those, top-p keeps an entry while the mass before it is below top_p, min-p keeps
 * p >= min_p * max p; an entry that both keep may be drawn.  The token is the first index, in the order of the vocabulary,
 * up to which the kept mass is above draw times the whole kept mass; its log-probability is among the kept entries.
 * temperature <= 0 takes the largest logit (the lowest index of equal ones).  k <= 0, top_p >= 1 and min_p <= 0 turn a
 * filter off; top_p <= 0 leaves the first entry, min_p >= 1 those that equal it.  draw is held to [0, 1).  A NaN logit or -inf is never
 * drawn, entries of +inf share the whole mass; a row of nothing else gives token -1 and log-probability -inf.  An entry
 * of 2^-44 of the largest mass or less counts for nothing, also where a filter keeps it.  A
 * parameter that is NaN turns its filter off (temperature: 0, draw: 0).  vocab <= 2^18, rows < 2^22.
 * Each parameter array holds one value per row, or a null pointer turns it off (temperature null: 1).  float32, k int32.
 */
typedef struct {
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
} fhe_ssm_sample_params;

/* logits: rows of vocab elements of `type`, row_stride elements apart.  tokens: int64[rows]; logprobs: float32[rows] or
 * null; draws: float32[rows]. */
int fhe_ssm_sample(uint32_t type, const void* logits, uint32_t rows, uint32_t vocab, int64_t row_stride,
                   const float* draws, const fhe_ssm_sample_params* params, int64_t* tokens, float* logprobs,
                   void* stream);

/* ---- layer norm ---------------------------------------------------------------------------------------------------
 *     y = (x - mean) rstd weight + bias,  rstd = 1 / sqrt(mean of (x - mean)^2 + eps)      over the channels of a row
 * channels <= 16384, rows < 2^31.  Rows are `type`, their strides in elements; weight and bias have `channels` elements of
 * weight_type, float32 or `type`, and null stands for 1 and 0.  mean and rstd (float32[rows], either may be null) are what the
 * backward pass takes.  out may be x; other overlaps are not allowed.  A row that holds a NaN or an infinity comes out NaN and
 * leaves the others alone.  Sums are float32: magnitudes of a row, and squares of its distances from the mean, have to sum to less
 * than 2^128, and with eps 0 squares below 2^-126 are lost. */
typedef struct {
    uint32_t type, weight_type; /* of x, out, dy and dx; of weight and bias */
    uint32_t rows, channels;
    float eps;
    int64_t x_stride, out_stride; /* out, backward dx */
    int64_t dy_stride;            /* backward only */
} fhe_ssm_layer_norm;

/* Device memory that a backward pass of these sizes needs for the weight's gradient (0: workspace may be null). */
int fhe_ssm_layer_norm_workspace(const fhe_ssm_layer_norm* a, size_t* bytes);

int fhe_ssm_layer_norm_forward(const fhe_ssm_layer_norm* a, const void* x, const void* weight, const void* bias, void* out,
                               float* mean, float* rstd, void* stream);

/* dx; dweight and dbias (float32[channels]) where they are not null, without rows zeros.  dx may be dy. */
int fhe_ssm_layer_norm_backward(const fhe_ssm_layer_norm* a, const void* dy, const void* x, const void* weight,
                                const float* mean, const float* rstd, void* dx, float* dweight, float* dbias,
                                void* workspace, size_t workspace_bytes, void* stream);

/* ---- gated linear recurrence --------------------------------------------------------------------------------------
 * Per lane and channel, with the state h in float32:
 *     a_t = sigmoid(z_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t,   out_t = h_t
 * lanes and tokens may be 0; tokens <= 2^24, channels <= 2^24, lanes * ceil(channels / 64) < 2^23.  Strides are in elements, in
 * the order lane, token, and may be any, except that rows of an output must not overlap; channels are contiguous.  States are
 * float32 [lanes][channels]: state_in null means zero, state_out null drops the new one, and the two may be the same buffer.
 * Outputs must overlap no input.  lengths as for linear attention: behind them nothing is read, outputs and gradients are zero.
 * What is not finite reaches its own channel of its own lane, from its token on, in the gradients back from it too. */
typedef struct {
    uint32_t type; /* of z, x, out and their gradients */
    uint32_t lanes, tokens, channels;
    int64_t z_stride[2], x_stride[2], out_stride[2];
    int64_t dout_stride[2], dz_stride[2], dx_stride[2]; /* backward only */
} fhe_ssm_gated_recurrence;

/* Device memory that a prompt or its backward pass of these sizes needs (0: workspace may be null), and that of what a prompt
 * saves for its backward pass. */
int fhe_ssm_gated_recurrence_workspace(const fhe_ssm_gated_recurrence* a, size_t* workspace_bytes, size_t* saved_bytes);

/* A prompt.  saved: null, or what the backward pass is given. */
int fhe_ssm_gated_recurrence_prompt(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const int32_t* lengths,
                                    const float* state_in, float* state_out, void* out, void* saved, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* From the gradients dout (null: zeros) and dstate_out (null: zeros) those of z, x and, where it is not null, state_in; z, x,
 * lengths, sizes and saved are the prompt's.  dstate_in may be dstate_out. */
int fhe_ssm_gated_recurrence_backward(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const int32_t* lengths,
                                      const void* saved, const void* dout, const float* dstate_out, void* dz, void* dx,
                                      float* dstate_in, void* workspace, size_t workspace_bytes, void* stream);

/* One token for every lane: the same with tokens = 1 and no lengths. */
int fhe_ssm_gated_recurrence_step(const fhe_ssm_gated_recurrence* a, const void* z, const void* x, const float* state_in,
                                  float* state_out, void* out, void* stream);

/* ---- embedding ----------------------------------------------------------------------------------------------------
 *     out_t = scale table[token_t]        dtable[v] = scale sum of dout_t over the t with token_t = v
 * tokens: int64 on the device; one outside [0, vocab) gives a row of zeros and adds to no gradient.  vocab <= 2^18, tokens <=
 * 2^25, channels <= 2^20.  The lookup takes any of the types for either side. */
typedef struct {
    uint32_t table_type, row_type; /* of the table and its gradient; of out and dout */
    uint32_t tokens, vocab, channels;
    float scale;
    int64_t table_stride, row_stride; /* elements from row to row; the table's gradient is contiguous */
} fhe_ssm_embedding;

int fhe_ssm_embedding_lookup(const fhe_ssm_embedding* a, const int64_t* tokens, const void* table, void* out, void* stream);

/* Device memory that the gradient needs (0 for few tokens: workspace may be null). */
int fhe_ssm_embedding_workspace(const fhe_ssm_embedding* a, size_t* bytes);

/* All of dtable (float32, or row_type) is written, or with `accumulate` the sums are added to what is there.  Sums are taken in
 * float32, in an order that the tokens decide, and rounded once: equal calls give equal results.  Other tokens among them may
 * change the last bits of a token's sum. */
int fhe_ssm_embedding_gradient(const fhe_ssm_embedding* a, const int64_t* tokens, const void* dout, void* dtable,
                               int accumulate, void* workspace, size_t workspace_bytes, void* stream);

/* ---- log-probabilities of given tokens ----------------------------------------------------------------------------
 * Per row of logits l, with p = softmax(l):
 *     logprob = log p[token],  entropy = - sum p log p,  the `top` largest logits' tokens and log-probabilities
 * Alternatives are in the order of falling logits, equal ones by rising index.  A token outside [0, vocab) has log-probability
 * 0 and its weight counts for nothing: a padded position.  A logit of -inf has probability 0; a row of nothing else has
 * entropy 0 and log-probability -inf.  A NaN or +inf makes its row's numbers NaN (and a gradient whose weights are not 0); it
 * leaves other rows alone.  NaN and -inf are no alternatives: where there are fewer than `top`, the rest is token -1 with
 * log-probability -inf.  vocab <= 2^18, rows < 2^22, top <= 32. */
typedef struct {
    uint32_t type;
    uint32_t rows, vocab, top;
    int64_t row_stride, gradient_stride; /* in elements */
} fhe_ssm_token_logprobs;

/* Device memory that the log-probabilities of these sizes need (0: workspace may be null). */
int fhe_ssm_token_logprobs_workspace(const fhe_ssm_token_logprobs* a, size_t* bytes);

/* tokens: int64[rows], null where no token is given.  logprobs, entropy: float32[rows], statistics: float32[rows][2], a row's
 * largest logit and the log of sum exp(l - largest); each may be null.  top_tokens int64[rows][top], top_logprobs
 * float32[rows][top], unless top is 0.  gradient, where it is not null: that of
 *     sum over rows of weights logprob + entropy_weights entropy          (float32[rows], null: 0)
 * with respect to the logits, in their type; it may be the logits' own buffer, with their stride. */
int fhe_ssm_token_logprobs_forward(const fhe_ssm_token_logprobs* a, const void* logits, const int64_t* tokens,
                                   float* logprobs, float* entropy, float* statistics, int64_t* top_tokens,
                                   float* top_logprobs, const float* weights, const float* entropy_weights, void* gradient,
                                   void* workspace, size_t workspace_bytes, void* stream);

/* The same gradient where its weights were not known before: from the statistics, and the entropy if it has weights. */
int fhe_ssm_token_logprobs_gradient(const fhe_ssm_token_logprobs* a, const void* logits, const int64_t* tokens,
                                    const float* statistics, const float* entropy, const float* weights,
                                    const float* entropy_weights, void* gradient, void* stream);

/* ---- AdamW --------------------------------------------------------------------------------------------------------
 * For every entry of every tensor, with g the gradient times *scale_at:
 *     m <- beta1 m + (1 - beta1) g,  v <- beta2 v + (1 - beta2) g^2,
 *     p <- p - lr (weight_decay p + m / (1 - beta1^step) / (sqrt(v / (1 - beta2^step)) + eps))
 * Parameters are float32; copy, where it is not null, receives them rounded to copy_type, for the products of the next pass.
 * With state_bits 32, first and second are m and v in float32.  With 8 they are m and sqrt(v) as 8-bit floats (a sign, 4 bits
 * of exponent with bias 7, 3 of mantissa), in blocks of 256 entries from the tensor's beginning; powers[block] has the powers of
 * two behind the codes of m and of the root, as their exponent plus 134, 255 for NaN.  Zeros are the beginning of all.  8-bit
 * states are rounded at random, by (seed, step, the tensor's place, the entry): equal calls give equal results.  A moment that
 * is not finite loses its entry, with 8 bits its block, whose parameters are NaN from the next step on.  A finite gradient whose
 * square overflows, above 1.8e19, stops its entry (v is infinite), with 8 bits it loses the block.
 * lr_at, step_at and scale_at, where they are not null, are read on the device in place of lr, step and 1, so that a recorded
 * step follows them; a step there that is below 1 changes nothing.  Tensors of no entries are passed over; one has less than
 * 2^32.  What is written (parameters, states, powers, copies) must not overlap.  eps >= 1e-30. */
typedef struct {
    uint32_t gradient_type, copy_type; /* copies are bf16 or f16 */
    uint32_t state_bits;               /* 32 or 8 */
    uint32_t step, seed;               /* steps count from 1 */
    float lr, eps;
    double beta1, beta2;
    const float* lr_at;
    const float* scale_at;
    const int32_t* step_at;
} fhe_ssm_adamw;

typedef struct {
    float* param;
    const void* gradient;
    void *first, *second;
    uint8_t* powers; /* [ceil(n / 256)][2], only with 8 bits */
    void* copy;
    uint64_t n;
    float weight_decay;
} fhe_ssm_adamw_tensor;

/* tensors: an array on the host, read before the call returns. */
int fhe_ssm_adamw_step(const fhe_ssm_adamw* a, uint32_t count, const fhe_ssm_adamw_tensor* tensors, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FHE_SSM_CLEAR_H */
