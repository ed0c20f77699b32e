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

#ifdef __cplusplus
}
#endif

#endif /* FHE_SSM_CLEAR_H */
